"""Sampling's workspace goes by what the call uses (CPU)."""

from __future__ import annotations

import ctypes

import pytest

from thundersync_amd import _lib

MB = 1 << 20


@pytest.mark.parametrize("rows, vocab, most", [
    (1, 151936, 0.01), (512, 151936, 1.0), (4096, 151936, 8), (4096, 1000, 1.0), (1 << 20, 151936, 8), (4096, 1 << 21, 90),
])
def test_without_filters(rows, vocab, most):
    """A slice's statistics and sums are 80 bytes."""
    assert 0 < _lib.require_library().ts_sample_workspace(rows, vocab, 0) <= most * MB


@pytest.mark.parametrize("vocab", [1, 1000, 50257, 151936, 1 << 21])
def test_with_filters(vocab):
    """A row's candidates and histogram shares, of at most about 128 MB however many rows, and never less than one
    row's."""
    lib = _lib.require_library()
    sizes = {rows: lib.ts_sample_workspace(rows, vocab, 1) for rows in
             (1, 2, 64, 100, 512, 1000, 2000, 2277, 2278, 4096, 4097, 5000, 100000, (1 << 31) - 1)}
    assert min(sizes.values()) == sizes[1] >= 4096 * 8 + 2048 * 12
    assert max(sizes.values()) <= 136 * MB and sizes[512] <= 52 * MB


def test_a_call_asks_for_what_it_uses():
    """On the host, before a launch: enough is accepted up to the next check, a byte less is refused."""
    lib = _lib.require_library()
    p = ctypes.c_void_p(16)
    for top_k, top_p, filters in ((0, 1.0, 0), (1, 1.0, 0), (100, 1.0, 0), (8, 1.0, 1), (0, 0.9, 1)):
        need = lib.ts_sample_workspace(7, 100, filters)
        args = lambda size: (p, 100, 7, 100, p, _lib.TS_F32, None, 1.0, None, top_k, None, top_p, None, 0.0, p, p, p, size,  # noqa: E731, E501
                             _lib.TS_BF16, None)
        assert lib.ts_sample(*args(need - 1)) == 1, (top_k, top_p)
        assert f"need {need}" in lib.ts_hip_last_error().decode(), (top_k, top_p)
