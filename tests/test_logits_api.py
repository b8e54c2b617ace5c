"""Refusals of the adjustment of logits, without a GPU."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from thundersync_amd import _lib
from thundersync_amd.logits import adjust_logits, pack_allowed

Z, H, I32 = torch.zeros(3, 70), torch.zeros(3, 5, dtype=torch.int64), torch.zeros(3, dtype=torch.int32)
A = torch.zeros(3, 3, dtype=torch.int32)


@pytest.mark.parametrize("logits, options, error, words", [
    (torch.zeros(5), {}, ValueError, r"logits must be \[B, V\]"),
    (torch.zeros(2, 0), {}, ValueError, r"logits must be \[B, V\]"),
    (torch.zeros(1, 1).expand(1, (1 << 21) + 1), {}, ValueError, "a vocabulary of at most"),
    (Z.double(), {}, TypeError, "bf16, fp16 or fp32 logits"),
    (torch.zeros(3, 70, requires_grad=True), {}, RuntimeError, "logits require grad"),
    (Z, {"repetition": 1.2}, ValueError, "penalties need a history"),
    (Z, {"presence": torch.zeros(3)}, ValueError, "penalties need a history"),
    (Z, {"lengths": I32}, ValueError, "are a history's"),
    (Z, {"history": H[:2]}, ValueError, r"history must be \[3, N\]"),
    (Z, {"history": H[:, 0]}, ValueError, r"history must be \[3, N\]"),
    (Z, {"history": H.float()}, TypeError, "history must be int64 or int32"),
    (Z, {"history": H, "lengths": I32[:2]}, ValueError, r"lengths must be \[3\]"),
    (Z, {"history": H, "lengths": I32.long()}, TypeError, "lengths must be int32"),
    (Z, {"history": H, "prompt_lengths": I32.long()}, TypeError, "prompt_lengths must be int32"),
    (Z, {"history": H, "repetition": 0.0}, ValueError, "repetition must be above 0"),
    (Z, {"history": H, "repetition": -1}, ValueError, "repetition must be above 0"),
    (Z, {"history": H, "repetition": 1e-60}, ValueError, "repetition must be above 0"),
    (Z, {"history": H, "repetition": "1"}, ValueError, "repetition must be a finite number"),
    (Z, {"history": H, "frequency": math.nan}, ValueError, "frequency must be a finite number"),
    (Z, {"history": H, "presence": 1e60}, ValueError, "presence must be a finite number"),
    (Z, {"history": H, "presence": torch.zeros(2)}, ValueError, r"presence must be \[3\]"),
    (Z, {"history": H, "presence": torch.zeros(3).double()}, TypeError, "presence must be float32"),
    (Z, {"bias": torch.zeros(3, 2)}, ValueError, "go together"),
    (Z, {"bias_ids": H}, ValueError, "go together"),
    (Z, {"bias_ids": H, "bias": torch.zeros(3, 4)}, ValueError, "bias must have the shape of bias_ids"),
    (Z, {"bias_ids": H, "bias": torch.zeros(3, 5).double()}, TypeError, "bias must be float32"),
    (Z, {"bias_ids": H.float(), "bias": torch.zeros(3, 5)}, TypeError, "bias_ids must be int64 or int32"),
    (Z, {"allowed": A[:, :2]}, ValueError, r"allowed must be \[M, 3\]"),
    (Z, {"allowed": A.long()}, TypeError, "allowed must be int32"),
    (Z, {"allowed": A[:2]}, ValueError, "a mask a row without allowed_rows"),
    (Z, {"allowed_rows": I32}, ValueError, "allowed_rows without allowed"),
    (Z, {"allowed": A, "allowed_rows": I32.long()}, TypeError, "allowed_rows must be int32"),
    (Z, {"allowed": A, "allowed_rows": I32[:2]}, ValueError, r"allowed_rows must be \[3\]"),
    (Z, {"out": torch.zeros(3, 69)}, ValueError, "out must be like logits"),
    (Z, {"out": torch.zeros(3, 70).half()}, ValueError, "out must be like logits"),
    (Z, {"out": torch.zeros(70, 3).t()}, ValueError, "out must have rows of their own"),
    (Z, {"out": torch.zeros(1, 70).expand(3, 70)}, ValueError, "out must have rows of their own"),
    (torch.zeros(300)[:210].view(3, 70), {}, RuntimeError, "on the GPU only"),
])
def test_refusals(logits, options, error, words):
    with pytest.raises(error, match=words):
        adjust_logits(logits, **options)


def test_an_output_that_overlaps_the_logits_otherwise_is_refused():
    x = torch.zeros(500)
    for out in (x[1:211].view(3, 70), x[70:280].view(3, 70)):
        with pytest.raises(ValueError, match="overlaps"):
            adjust_logits(x[:210].view(3, 70), out=out)
    with pytest.raises(RuntimeError, match="on the GPU only"):
        adjust_logits(x[:210].view(3, 70), out=x[:210].view(3, 70))
    with pytest.raises(RuntimeError, match="on the GPU only"):
        adjust_logits(x[:210].view(3, 70), out=x[210:420].view(3, 70))


def test_pack_allowed():
    mask = torch.zeros(2, 65, dtype=torch.bool)
    mask[0, [0, 31, 32, 64]] = True
    mask[1] = True
    assert pack_allowed(mask).tolist() == [[1 - (1 << 31), 1, 1], [-1, -1, 1]]
    for bad in (mask[0], mask.int()):
        with pytest.raises(ValueError, match="a bool mask"):
            pack_allowed(bad)


def test_the_c_entry_refuses():
    lib, p = _lib.require_library(), ctypes.c_void_p(4096)
    good = dict(z=p, ld=70, rows=3, vocab=70, h=p, ldh=5, w=5, n=None, pr=None, r=None, ra=1.0, f=None, fa=0.0, pp=None,
                pa=0.0, bi=None, ldbi=0, b=None, ldb=0, nb=0, a=None, lda=0, ar=None, m=0, idb=8, o=p, ldo=70, dt=0, st=None)
    for change, words in (({"dt": 3}, "dtype 3"), ({"vocab": 0}, "bad shape"), ({"rows": -1}, "bad shape"),
                          ({"vocab": (1 << 21) + 1}, "bad shape"), ({"ldo": 69}, "bad shape"), ({"idb": 2}, "ids of 2 bytes"),
                          ({"w": -1}, "bad lists"), ({"nb": -1}, "bad lists"), ({"nb": 3}, "null pointer"),
                          ({"z": None}, "null pointer"), ({"o": None}, "null pointer"),
                          ({"rows": 1 << 30}, "grid too large"), ({"ra": 0.0}, "penalty"), ({"ra": math.nan}, "penalty")):
        assert lib.ts_adjust_logits(*(good | change).values()) == 1, change
        assert words in lib.ts_hip_last_error().decode(), (change, lib.ts_hip_last_error())
