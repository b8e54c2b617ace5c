"""Refusals of distillation, embedding and sampling, and the embedding swap, without a GPU."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from thundersync_amd import _lib, embedding, fused_distill, sampling


def _distill_args(n=4, d=8, v=16, k=3):
    return [torch.zeros(n, d), torch.zeros(v, d), torch.zeros(n, k, dtype=torch.int64), torch.zeros(n, k)]


@pytest.mark.parametrize("change, error, words", [
    ({0: torch.zeros(8)}, ValueError, r"hidden must be \[N, D\]"),
    ({1: torch.zeros(16, 9)}, ValueError, "does not match hidden dim 8"),
    ({2: torch.zeros(5, 3, dtype=torch.int64)}, ValueError, "one row per hidden row"),
    ({2: torch.zeros(4, dtype=torch.int64)}, ValueError, "one row per hidden row"),
    ({3: torch.zeros(4, 2)}, ValueError, "must have the shape of teacher_ids"),
    ({2: torch.zeros(4, 0, dtype=torch.int64), 3: torch.zeros(4, 0)}, ValueError, "1 to 1024 teacher logits"),
    ({2: torch.zeros(4, 1025, dtype=torch.int64), 3: torch.zeros(4, 1025)}, ValueError, "1 to 1024 teacher logits"),
    ({1: torch.zeros(0, 8)}, ValueError, "an empty head"),
    ({2: torch.zeros(4, 3)}, TypeError, "teacher_ids must be int64 or int32"),
    ({3: torch.zeros(4, 3, dtype=torch.int32)}, TypeError, "teacher_logits must be"),
    ({}, RuntimeError, "runs on the GPU only"),
])
def test_distill_refusals(change, error, words):
    args = _distill_args()
    for i, t in change.items():
        args[i] = t
    with pytest.raises(error, match=words):
        fused_distill.fused_distill(*args)


@pytest.mark.parametrize("temperature", [0.0, -1.0, math.inf, math.nan, "1", torch.tensor(1.0)])
def test_distill_temperature(temperature):
    with pytest.raises(ValueError, match="temperature must be a positive number"):
        fused_distill.fused_distill(*_distill_args(), temperature=temperature)


@pytest.mark.parametrize("ids, weight, options, error, words", [
    (torch.zeros(3, dtype=torch.int64), torch.zeros(8), {}, ValueError, r"weight must be \[V, D\]"),
    (torch.zeros(3), torch.zeros(8, 4), {}, TypeError, "ids must be int64 or int32"),
    (torch.zeros(3, dtype=torch.int64), torch.zeros(8, 4), {"scale": math.inf}, ValueError, "scale must be"),
    (torch.zeros(3, dtype=torch.int64), torch.zeros(8, 4), {"padding_idx": 8}, ValueError, "padding_idx 8"),
    (torch.zeros(3, dtype=torch.int64), torch.zeros(8, 4), {"padding_idx": -1}, ValueError, "padding_idx -1"),
    (torch.zeros(3, dtype=torch.int64), torch.zeros(8, 4), {}, RuntimeError, "runs on the GPU only"),
])
def test_embedding_refusals(ids, weight, options, error, words):
    with pytest.raises(error, match=words):
        embedding.embedding(ids, weight, **options)


@pytest.mark.parametrize("logits, uniform, options, error, words", [
    (torch.zeros(8), torch.zeros(1), {}, ValueError, r"logits must be \[B, V\]"),
    (torch.zeros(2, 0), torch.zeros(2), {}, ValueError, r"logits must be \[B, V\]"),
    (torch.zeros(2, 8), torch.zeros(3), {}, ValueError, "one number per row"),
    (torch.zeros(1, 1).expand(1, (1 << 21) + 1), torch.zeros(1), {}, ValueError, "a vocabulary of at most"),
    (torch.zeros(2, 8, dtype=torch.float64), torch.zeros(2), {}, TypeError, "bf16, fp16 or fp32 logits"),
    (torch.zeros(2, 8), torch.zeros(2, dtype=torch.float16), {}, TypeError, "uniform must be fp32 or fp64"),
    (torch.zeros(2, 8), torch.zeros(2), {"temperature": -0.1}, ValueError, "temperature must be a finite number"),
    (torch.zeros(2, 8), torch.zeros(2), {"temperature": math.inf}, ValueError, "temperature must be a finite number"),
    (torch.zeros(2, 8), torch.zeros(2), {"top_p": math.nan}, ValueError, "top_p must be a finite number"),
    (torch.zeros(2, 8), torch.zeros(2), {"top_k": 1.5}, ValueError, "top_k must be a whole number"),
    (torch.zeros(2, 8), torch.zeros(2), {"top_k": -1}, ValueError, "top_k must be a finite number"),
    (torch.zeros(2, 8), torch.zeros(2), {"min_p": torch.zeros(3)}, ValueError, "one value per row"),
    (torch.zeros(2, 8), torch.zeros(2), {"min_p": torch.zeros(2, dtype=torch.float64)}, TypeError, "min_p per row"),
    (torch.zeros(2, 8), torch.zeros(2), {"top_k": torch.zeros(2)}, TypeError, "top_k per row must be torch.int32"),
    (torch.zeros(2, 8), torch.zeros(2), {}, RuntimeError, "runs on the GPU only"),
])
def test_sampling_refusals(logits, uniform, options, error, words):
    with pytest.raises(error, match=words):
        sampling.sample_tokens(logits, uniform, **options)


def test_c_entries_refuse_without_a_device():
    lib = _lib.require_library()
    p = ctypes.c_void_p(16)  # never read: every call below is refused on the host
    bf16, f32 = _lib.TS_BF16, _lib.TS_F32
    calls = {
        "ts_distill_teacher": [
            (p, p, 4, f32, 2, 1025, 100, 1.0, p, p, 1025, p, bf16, None),
            (p, p, 4, f32, 2, 4, 100, 0.0, p, p, 4, p, bf16, None),
            (p, p, 4, f32, 2, 4, 100, math.nan, p, p, 4, p, bf16, None),
            (None, p, 4, f32, 2, 4, 100, 1.0, p, p, 4, p, bf16, None),
        ],
        "ts_embedding_fwd": [
            (p, 2, p, 3, 10, 4, 1.0, p, bf16, None),
            (p, 2, p, 4, 10, 4, 1.0, p, _lib.TS_F64, None),
            (None, 2, p, 4, 10, 4, 1.0, p, bf16, None),
        ],
        "ts_embedding_bwd": [
            (p, 2, p, 4, 10, 4, -1, 1.0, ctypes.c_void_p(8), p, 1 << 20, bf16, None),
            (p, 2, p, 4, 1 << 31, 4, -1, 1.0, p, p, 1 << 20, bf16, None),
        ],
        "ts_sample": [
            (p, 8, 2, (1 << 21) + 1, p, f32, None, 1.0, None, 0, None, 1.0, None, 0.0, p, p, p, 1 << 20, bf16, None),
            (p, 8, 2, 8, p, f32, None, math.nan, None, 0, None, 1.0, None, 0.0, p, p, p, 1 << 20, bf16, None),
            (p, 8, 2, 8, p, f32, None, 1.0, None, 0, None, 1.0, None, 0.0, p, p, p, 16, bf16, None),
            (p, 8, 2, 8, None, f32, None, 1.0, None, 0, None, 1.0, None, 0.0, p, p, p, 1 << 20, bf16, None),
        ],
    }
    for name, cases in calls.items():
        for args in cases:
            assert getattr(lib, name)(*args) == 1, (name, args)
            assert name in lib.ts_hip_last_error().decode()


def test_embedding_swap_keeps_the_parameter_and_torchs_cpu_forward():
    class Tied(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.table = torch.nn.Embedding(10, 4, padding_idx=1)
            self.scaled = torch.nn.Embedding(10, 4, scale_grad_by_freq=True)
            self.head = torch.nn.Linear(4, 10, bias=False)
            self.head.weight = self.table.weight

    model = Tied().eval()
    weight, ids = model.table.weight, torch.tensor([[1, 2], [3, 9]])
    want = model.table(ids)
    assert embedding.use_hip_embedding(model) == 1
    assert type(model.table) is embedding.HipEmbedding and type(model.scaled) is torch.nn.Embedding
    assert model.table.weight is weight is model.head.weight and not model.table.training
    assert model.table.padding_idx == 1 and torch.equal(model.table(ids), want)
    assert embedding.use_hip_embedding(model) == 0
    assert list(model.state_dict()) == list(Tied().state_dict())
