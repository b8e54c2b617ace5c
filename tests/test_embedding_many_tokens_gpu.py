"""More tokens than a launch has work-groups along one axis (2^32 threads), and those a gradient refuses."""

from __future__ import annotations

import ctypes

import pytest
import torch

from thundersync_amd import _lib
from thundersync_amd.embedding import embedding, embedding_backward


def test_a_gradient_of_too_many_tokens_is_refused():
    lib = _lib.require_library()
    p = ctypes.c_void_p(16)  # never read
    for n in (1 << 28, (1 << 31) - 1):
        assert lib.ts_embedding_bwd(p, n, p, 8, 10, 8, -1, 1.0, p, p, 1 << 60, _lib.TS_BF16, None) == 1
        assert "bad shape" in lib.ts_hip_last_error().decode()


@pytest.mark.gpu
def test_rows_past_one_launch(cuda):
    """2^24 + 5 tokens of rows that take a work-group each: 4.3 GB."""
    n, d, v = (1 << 24) + 5, 129, 7
    print(f"embedding of {n} tokens", flush=True)
    table = torch.randn(v, d, generator=torch.Generator(device=cuda).manual_seed(0), device=cuda).bfloat16()
    ids = torch.arange(n, device=cuda) % v
    out = embedding(ids, table)
    for part in (slice(0, 1000), slice((1 << 23) - 500, (1 << 23) + 500), slice(n - 1000, n)):
        assert torch.equal(out[part], table[ids[part]])
    grad = embedding_backward(ids, torch.ones(1, 1, dtype=torch.float32, device=cuda).expand(n, 1), v)
    assert torch.equal(grad[:, 0].long(), torch.bincount(ids, minlength=v))
