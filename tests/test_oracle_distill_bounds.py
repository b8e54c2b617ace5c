"""The distillation oracle's bound on a loss is narrow enough to see a lost vocabulary tile (CPU)."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import distill


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_tile_left_out_or_taken_twice_shows(dtype):
    """At the sizes of the GPU test over a whole vocabulary: the loss moves by what the tile of 256 tokens (the last has
    128) adds to the sum of exponentials, in every row by more than the bound."""
    n, d, v, k = 2, 1024, 151936, 5
    g = torch.Generator().manual_seed(0)
    h = torch.randn(n, d, generator=g).to(dtype)
    w = (torch.randn(v, d, generator=g) * 0.05).to(dtype)
    ids = torch.randint(0, v, (n, k), generator=g)
    ref = distill.distill(h, w, ids, torch.randn(n, k, generator=g) * 2, torch.ones(n))
    bound = distill.bounds(ref, dtype, k)["loss"]
    assert bound.max() <= 2.5e-4
    tiles = torch.nn.functional.pad(ref["q"], (0, -v % 256)).view(n, -1, 256).sum(dim=2)
    assert tiles.shape[1] == 594
    for change in (torch.log1p(-tiles), torch.log1p(tiles)):  # of the row's loss: its slots' p add up to 1
        assert (change[:, -1].abs() > bound).all(), (change[:, -1], bound)
        assert (change.abs() > bound[:, None]).all(), (change.abs().min(), bound)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_the_exact_types(dtype):
    n, d, v, k = 2, 256, 32003, 5
    g = torch.Generator().manual_seed(0)
    h = torch.randn(n, d, generator=g).to(dtype)
    w = (torch.randn(v, d, generator=g) * 0.05).to(dtype)
    ref = distill.distill(h, w, torch.randint(0, v, (n, k), generator=g), torch.randn(n, k, generator=g), torch.ones(n))
    bound = distill.bounds(ref, dtype, k)["loss"]
    assert bound.max() <= (5e-4 if dtype == torch.float32 else 1e-12)
    assert math.isfinite(bound.max())
