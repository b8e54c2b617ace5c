"""Calls whose launches would take 2^32 threads along an axis, which wrap without an error, are refused (CPU)."""

from __future__ import annotations

import ctypes

import pytest

from thundersync_amd import _lib

P = ctypes.c_void_p(4096)  # never read: refused on the host
BF16, F32 = _lib.TS_BF16, _lib.TS_F32
MANY, SPACE = 1 << 23, 1 << 62


@pytest.mark.parametrize("name, args, words", [
    # tiles of 256 rows x 256 tokens, 512 threads each
    ("ts_logprob_fwd", (P, 8, P, 8, P, 4_000_000, 8, 151936, P, None, P, P, SPACE, BF16, None), "grid too large"),
    ("ts_logprob_fwd", (P, 8, P, 8, P, 1 << 28, 8, 8, P, None, P, P, SPACE, BF16, None), "grid too large"),
    ("ts_logprob_dlogits", (P, 8, P, 8, P, P, None, P, None, 4_000_000, 8, 151936, P, 151936, BF16, None),
     "grid too large"),
    ("ts_logprob_grad_weight_block", (P, 1 << 24, P, 1 << 20, 4, (1 << 20) - 8, 1 << 24, P, 1 << 20, 1, None, 0, BF16,
                                      None), "grid too large"),
    ("ts_distill_fwd", (P, 8, P, 8, 4_000_000, 8, 151936, 1.0, P, P, P, 8, 8, P, P, P, None, 0, None, P, SPACE, BF16,
                        None), "grid too large"),
    ("ts_distill_dlogits", (P, 8, P, 8, 4_000_000, 8, 151936, 1.0, P, P, P, 8, 8, P, P, P, P, 151936, BF16, None),
     "grid too large"),
    # a work-group a row
    ("ts_distill_teacher", (P, P, 8, F32, MANY, 8, 100, 1.0, P, P, 8, P, BF16, None), "bad shape"),
    ("ts_distill_fwd", (P, 8, P, 8, MANY, 8, 8, 1.0, P, P, P, 8, 8, P, P, P, None, 0, None, P, SPACE, BF16, None),
     "bad shape"),
    ("ts_distill_fwd_exact", (P, 8, MANY, 8, 1.0, P, P, P, 8, 8, P, P, P, F32, None), "bad shape"),
    ("ts_distill_finish", (P, 8, P, MANY, 8, 1.0, P, P, P, 8, 8, P, P, P, P, 8, BF16, None), "bad shape"),
    ("ts_distill_softmax", (P, 8, P, P, MANY, 8, P, 8, 8, P, BF16, None), "bad shape"),
    ("ts_distill_slots", (P, P, P, 8, MANY, 8, 1.0, P, P, P, 8, 8, P, BF16, None), "bad shape"),
    ("ts_distill_rows", (P, 8, P, MANY, 8, P, BF16, None), "bad shape"),
    ("ts_distill_scale", (P, P, P, MANY, 8, 1.0, P, BF16, None), "bad shape"),
])
def test_refused(name, args, words):
    lib = _lib.require_library()
    assert getattr(lib, name)(*args) == 1, name
    assert words in lib.ts_hip_last_error().decode()
