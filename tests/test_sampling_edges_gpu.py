"""Sampling at the ends of its options."""

from __future__ import annotations

import math

import pytest
import torch

from thundersync_amd.sampling import sample_tokens

pytestmark = pytest.mark.gpu


def test_a_rows_nan_options_filter_nothing(cuda):
    """As a NaN top_p always did, so a NaN min_p: the token is the unfiltered one."""
    g = torch.Generator(device=cuda).manual_seed(0)
    z = torch.randn(6, 1000, generator=g, device=cuda)
    u = torch.rand(6, generator=g, device=cuda)
    want = sample_tokens(z, u)
    nan = torch.full((6,), math.nan, device=cuda)
    for options in ({"min_p": nan}, {"top_p": nan}, {"min_p": nan, "top_p": nan}):
        got = sample_tokens(z, u, **options)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), list(options)
    half = torch.full((6,), 0.5, device=cuda)
    want = sample_tokens(z, u, top_p=half)
    got = sample_tokens(z, u, top_p=half, min_p=nan)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
