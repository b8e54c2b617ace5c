"""Sampling at the ends of its options."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import sampling as ref
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


@pytest.mark.parametrize("temperature", [1e30, 1e292, 1.7e308])
@pytest.mark.parametrize("options", [{}, {"top_p": 0.9}, {"top_k": 7}, {"min_p": 0.5}])
def test_infinite_logits_at_any_temperature(cuda, temperature, options):
    """A logit below an infinite one has no weight, however hot the row; among finite ones everything is even (0.1 in
    fp32 is above a tenth, 0.9 below nine)."""
    z = torch.zeros(2, 3000, device=cuda)
    z[0, 17] = z[0, 2900] = math.inf
    z[1] = torch.arange(3000, device=cuda) % 7
    for u, first, second in ((0.1, 17, 300), (0.9, 2900, 2699)):
        tokens, logprobs = sample_tokens(z, torch.full((2,), u, device=cuda), temperature=temperature, **options)
        assert tokens[0] == first and abs(logprobs[0].item() - math.log(0.5)) <= 2.0 ** -24
        if not options:
            assert tokens[1] == second and abs(logprobs[1].item() + math.log(3000)) <= 2.0 ** -20


@pytest.mark.parametrize("options", [{}, {"top_p": 0.9, "top_k": 40}])
def test_rows_of_several_sets(cuda, options):
    """Rows past one set of launches, the last set shorter: each row's token is its own."""
    g = torch.Generator(device=cuda).manual_seed(3)
    z = torch.randn(5003, 3000, generator=g, device=cuda)
    u = torch.rand(5003, generator=g, device=cuda)
    got = sample_tokens(z, u, **options)
    for part in (slice(0, 5), slice(1666, 1672), slice(2500, 2504), slice(4990, 5003)):
        want = sample_tokens(z[part], u[part], **options)
        assert torch.equal(got[0][part], want[0]) and torch.equal(got[1][part], want[1])
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    sample_tokens(z, u, **options)
    assert torch.cuda.max_memory_allocated() - before <= (136 << 20 if options else 8 << 20)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("options", [{"temperature": 5.0, "top_p": 0.9}, {"temperature": 5.0, "top_k": 9000},
                                     {"temperature": 3.0, "top_k": 20000, "top_p": 0.8, "min_p": 0.01}])
def test_masks_of_the_lowest_finite_value(cuda, dtype, options):
    """Such a mask stretches the row's range to the type's, and close logits then share a few bins, more of them than
    are sorted at once: the same tokens as with masks of -inf."""
    g = torch.Generator(device=cuda).manual_seed(1)
    z = (0.3 * torch.randn(3, 40001, generator=g, device=cuda)).to(dtype)
    masked = torch.rand(3, 40001, generator=g, device=cuda) < 0.2
    u = torch.rand(3, generator=g, device=cuda, dtype=torch.float64)
    want = sample_tokens(z.masked_fill(masked, -math.inf), u, **options)
    low = z.masked_fill(masked, torch.finfo(dtype).min)
    got = sample_tokens(low, u, **options)
    assert torch.equal(got[0], want[0])
    for i in range(3):
        token, logprob = ref.sample(low[i].double().cpu().numpy(), float(u[i]), **options)
        assert got[0][i] == token and abs(got[1][i].item() - logprob) <= 2.0 ** -23 * max(1.0, abs(logprob))
