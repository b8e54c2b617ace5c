"""Inputs of distillation and of the fused logprob that are valid as torch hands them over."""

from __future__ import annotations

import math

import pytest
import torch

from thundersync_amd.fused_distill import fused_distill
from thundersync_amd.fused_logprob import fused_logprob

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def inputs(cuda, n, d, v, k, dtype, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    h = torch.randn(n, d, generator=g, device=cuda).to(dtype)
    w = (torch.randn(v, d, generator=g, device=cuda) * 0.1).to(dtype)
    ids = torch.stack([torch.randperm(v, generator=g, device=cuda)[:k] for _ in range(n)])
    return h, w, ids, torch.randn(n, k, generator=g, device=cuda) * 2


def both(h, w, ids, teacher):
    """Loss and gradients with a trainable head."""
    h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
    loss = fused_distill(h, w, ids, teacher)
    return [loss.detach(), *torch.autograd.grad(loss.sum(), (h, w))]


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_one_row_of_a_teacher(cuda, dtype):
    """A column seen as a row has a row stride of 1, and one row of an expanded teacher one of 0: torch calls both
    contiguous."""
    h, w, ids, teacher = inputs(cuda, 1, 32, 300, 6, dtype)
    want = both(h, w, ids, teacher)
    column = teacher.reshape(6, 1).T
    assert column.stride() == (1, 1)
    expanded = teacher.expand(4, 6)[:1].as_strided((1, 6), (0, 1))
    for t in (column, expanded):
        assert all(torch.equal(a, b) for a, b in zip(both(h, w, ids, t), want))
    assert all(torch.equal(a, b) for a, b in zip(both(h, w, ids.reshape(6, 1).T, teacher), want))


@pytest.mark.parametrize("absent_id", [300, 1 << 40])
def test_checked_ids_pass_absent_slots(cuda, absent_id, monkeypatch):
    """THUNDERSYNC_CHECK_TARGETS looks at present slots: an absent one may name any token."""
    h, w, ids, teacher = inputs(cuda, 3, 32, 300, 6, BF16)
    teacher[1, 4] = -math.inf
    want = both(h, w, ids, teacher)
    ids[1, 4] = absent_id
    monkeypatch.setenv("THUNDERSYNC_CHECK_TARGETS", "1")
    assert all(torch.equal(a, b) for a, b in zip(both(h, w, ids, teacher), want))
    ids[2, 0] = absent_id
    with pytest.raises(ValueError, match=rf"target\[2\] = {absent_id} is outside the vocabulary"):
        fused_distill(h, w, ids, teacher)


def off_border(t):
    """``t`` contiguous, two bytes past a 16-byte border."""
    flat = torch.empty(t.numel() + 8, dtype=t.dtype, device=t.device)[1 : t.numel() + 1]
    out = flat.view(t.shape)
    out.copy_(t)
    assert out.is_contiguous() and out.data_ptr() % 16
    return out


def one_row_of(t, width):
    """The one row of ``t`` in a buffer whose rows are ``width`` apart."""
    buffer = torch.zeros(2, width, dtype=t.dtype, device=t.device)
    buffer[0, : t.shape[1]] = t[0]
    return buffer[:1, : t.shape[1]]


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_rows_off_a_16_byte_border(cuda, dtype):
    h, w, ids, teacher = inputs(cuda, 9, 64, 300, 6, dtype)
    want = both(h, w, ids, teacher)
    assert all(torch.equal(a, b) for a, b in zip(both(off_border(h), off_border(w), ids, teacher), want))
    frozen = fused_distill(off_border(h), off_border(w), ids, teacher)
    assert torch.equal(frozen, want[0])


def logprob(h, w, target):
    h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
    lp = fused_logprob(h, w, target)
    return [lp.detach(), *torch.autograd.grad(lp.sum(), (h, w))]


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_logprob_rows_off_a_16_byte_border(cuda, dtype):
    h, w, ids, _ = inputs(cuda, 9, 64, 300, 1, dtype)
    target = ids[:, 0].contiguous()
    want = logprob(h, w, target)
    assert all(torch.equal(a, b) for a, b in zip(logprob(off_border(h), off_border(w), target), want))
    want = logprob(h[:1], w, target[:1])
    assert all(torch.equal(a, b) for a, b in zip(logprob(one_row_of(h, 131), w, target[:1]), want))


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_one_row_of_wider_rows(cuda, dtype):
    h, w, ids, teacher = inputs(cuda, 1, 64, 300, 6, dtype)
    want = both(h, w, ids, teacher)
    assert all(torch.equal(a, b) for a, b in zip(both(one_row_of(h, 131), w, ids, teacher), want))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("d", [64, 50])
def test_logprob_of_repeated_rows(cuda, dtype, d):
    """One hidden row for every target, and a head of one row repeated: expanded tensors."""
    h, w, ids, _ = inputs(cuda, 9, d, 300, 1, dtype)
    target = ids[:, 0].contiguous()
    want = logprob(h[:1].expand(9, d).contiguous(), w, target)
    assert all(torch.equal(a, b) for a, b in zip(logprob(h[:1].expand(9, d), w, target), want))
    one = w[:1].expand(300, d)
    want = logprob(h, one.contiguous(), target)
    assert all(torch.equal(a, b) for a, b in zip(logprob(h, one, target), want))
