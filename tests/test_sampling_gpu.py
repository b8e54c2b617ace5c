"""Sampling against the fp64 oracle: the same tokens, logprobs within fp32's rounding.

A token could differ only where u times the total comes within the rounding of 64-bit sums of a step of the running
sum; the inputs' distances are checked to be far above it (``oracle.sampling.border_distance``)."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import sampling as ref
from thundersync_amd.sampling import sample_tokens

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def per_row(options, i):
    return {k: (float(x[i]) if isinstance(x, torch.Tensor) else x) for k, x in options.items()}


def check(cuda, z, u, **options):
    on_gpu = {k: x.to(cuda) if isinstance(x, torch.Tensor) else x for k, x in options.items()}
    tokens, logprobs = sample_tokens(z.to(cuda) if not z.is_cuda else z, u.to(cuda), **on_gpu)
    assert tokens.dtype == torch.int64 and logprobs.dtype == torch.float32
    tokens, logprobs = tokens.cpu().tolist(), logprobs.cpu().tolist()
    rows = z.detach().cpu().double().numpy()
    for i in range(len(rows)):
        o = per_row(options, i)
        o["top_k"] = int(o.get("top_k", 0))
        want, lp = ref.sample(rows[i], float(u[i]), **o)
        assert tokens[i] == want, f"row {i} {o} u={float(u[i])}: token {tokens[i]}, want {want}"
        if math.isnan(lp):
            assert math.isnan(logprobs[i])
        else:
            # fp64 sums of up to 2^21 weights (2^-30 at worst), then one rounding to fp32
            assert abs(logprobs[i] - lp) <= 2.0 ** -24 * abs(lp) + 2.0 ** -30, (i, logprobs[i], lp)


def logits(b, v, dtype, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(b, v, generator=g) * spread
    z[:, ::5] -= 3.0
    return z.to(dtype), torch.rand(b, generator=g)


MODES = {
    "none": {},
    "temperature": {"temperature": 0.3},
    "hot": {"temperature": 50.0},
    "top_k": {"top_k": 50},
    "top_k_most": {"top_k": 900, "temperature": 2.0},
    "top_p": {"top_p": 0.9},
    "top_p_small": {"top_p": 1e-6},
    "top_p_zero": {"top_p": 0.0},
    "top_p_most": {"top_p": 0.9999, "temperature": 3.0},
    "min_p": {"min_p": 0.05},
    "min_p_one": {"min_p": 1.0},
    "all": {"temperature": 0.8, "top_k": 200, "top_p": 0.9, "min_p": 0.01},
    "k_then_p": {"top_k": 40, "top_p": 0.5},
    "greedy": {"temperature": 0.0},
    "one": {"top_k": 1},
}


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("b, v", [(3, 1), (4, 2), (5, 7), (16, 1000), (6, 8193), (3, 50257)])
def test_tokens_and_logprobs(cuda, b, v, dtype, mode):
    print(f"sample b={b} v={v} {dtype} {mode}", flush=True)
    z, u = logits(b, v, dtype, seed=b + v)
    check(cuda, z, u, **MODES[mode])


@pytest.mark.parametrize("b, v, dtype", [(64, 3001, BF16), (7, 151936, BF16), (40, 20000, FP32), (33, 50257, FP16)])
def test_options_per_row(cuda, b, v, dtype):
    print(f"sample per row b={b} v={v} {dtype}", flush=True)
    z, u = logits(b, v, dtype, seed=b * v)
    g = torch.Generator().manual_seed(1)
    rand = lambda: torch.rand(b, generator=g)  # noqa: E731
    check(cuda, z, u, temperature=torch.where(rand() < 0.1, 0.0, 0.3 + rand()),
          top_k=torch.where(rand() < 0.4, 0, torch.randint(1, v + 10, (b,), generator=g)).int(),
          top_p=torch.where(rand() < 0.4, 1.0, rand()), min_p=torch.where(rand() < 0.4, 0.0, rand() * 0.2))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("v", [64, 5000, 20000, 70001])
def test_equal_logits(cuda, v, dtype):
    """Rows of one value, of two values, of few: the border falls among equal logits, which are kept by index."""
    print(f"sample equal logits v={v} {dtype}", flush=True)
    g = torch.Generator().manual_seed(v)
    z = torch.stack([torch.zeros(v), torch.randint(0, 2, (v,), generator=g).float(),
                     torch.randint(0, 5, (v,), generator=g) * 0.25, torch.full((v,), -3.0e38 if dtype == FP32 else -3.0e38)])
    z[3, v // 2] = -2.0e38
    z = z.to(dtype)
    for u in (0.0, 0.123, 0.77, 1.0 - 2.0 ** -24):
        us = torch.full((4,), u)
        for options in ({"top_k": 17}, {"top_k": v // 2 + 3}, {"top_p": 0.4999}, {"top_p": 0.77, "top_k": v // 3 + 1},
                        {"min_p": 0.5}, {}):
            check(cuda, z, us, **options)


def test_equal_logits_at_an_exact_border(cuda):
    """p times the total is the running sum itself: what is before an element has to be below it to keep it."""
    z = torch.zeros(3, 1024)
    for p in (0.5, 0.25, 0.75):
        check(cuda, z, torch.tensor([0.0, 0.5, 0.9999]), top_p=p)
    tokens, _ = sample_tokens(torch.zeros(1, 1024, device=cuda), torch.tensor([0.9999999], device=cuda), top_p=0.5)
    assert int(tokens) == 511


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_masked_and_extreme_logits(cuda, dtype):
    """-inf, the type's lowest value, infinities, NaN, both zeros."""
    print(f"sample extremes {dtype}", flush=True)
    low, inf, nan = torch.finfo(dtype).min, math.inf, math.nan
    base = torch.randn(12, 600, generator=torch.Generator().manual_seed(0))
    base[0] = -inf
    base[1], base[1, 333] = -inf, -5.0
    base[2] = low
    base[3], base[3, 7] = low, 1.0
    base[4, 100] = nan
    base[5], base[5, 599] = -inf, nan
    base[6, 5] = base[6, 400] = inf
    base[7, ::2] = -inf
    base[8] = 0.0
    base[8, ::3] = -0.0
    base[9] = torch.finfo(dtype).max
    base[10, 3], base[10, 4] = torch.finfo(dtype).max, low
    base[11] = inf
    z = base.to(dtype)
    for options in ({}, {"top_k": 5}, {"top_p": 0.7}, {"min_p": 0.3}, {"top_k": 300, "top_p": 0.9}, {"top_k": 599},
                    {"temperature": 0.0}, {"temperature": 1e-30, "top_p": 0.9}, {"temperature": 1e30, "top_p": 0.5}):
        for u in (0.0, 0.4, 0.999999):
            check(cuda, z, torch.full((12,), u), **options)


def test_random_numbers_outside_their_range_draw_the_last(cuda):
    z = torch.tensor([[0.0, 1.0, -math.inf], [2.0, 0.0, 0.5]], device=cuda)
    for u in (1.0, 1.5, math.nan, math.inf):
        tokens, logprobs = sample_tokens(z, torch.full((2,), u, device=cuda))
        assert tokens.tolist() == [1, 2] and logprobs.isfinite().all()
    assert sample_tokens(z, torch.full((2,), -1.0, device=cuda))[0].tolist() == [0, 0]
    wide = torch.full((1, 30000), -math.inf, device=cuda)
    wide[0, 20000:20002] = 0.0
    for u, want in ((-1.0, 20000), (0.0, 20000), (2.0, 20001), (math.nan, 20001)):
        for options in ({}, {"top_p": 0.9}, {"top_k": 7}, {"min_p": 0.5}):
            assert int(sample_tokens(wide, torch.full((1,), u, device=cuda), **options)[0]) == want


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_strides_and_alignment(cuda, dtype):
    """Row strides, rows that start off a 16-byte border, columns apart, a repeated row, fp64 random numbers."""
    z, u = logits(9, 1234, dtype, seed=5)
    flat = torch.zeros(9 * 1301 + 5, dtype=dtype, device=cuda)
    for off in range(4):
        view = flat[off : off + 9 * 1301].view(9, 1301)[:, 3 : 3 + 1234]
        view.copy_(z)
        for options in ({}, {"top_p": 0.8, "top_k": 100}):
            check(cuda, view, u, **options)
    check(cuda, z.to(cuda).T.contiguous().T, u, top_k=30)
    check(cuda, z[:1].to(cuda).expand(9, 1234), u, top_p=0.9)
    check(cuda, z, torch.rand(9, dtype=torch.float64, generator=torch.Generator().manual_seed(1)))
    assert sample_tokens(torch.zeros(0, 5, device=cuda), torch.zeros(0, device=cuda))[0].shape == (0,)


def test_per_row_values_that_are_no_options(cuda):
    """What the documentation says of per-row values that a number would be refused for."""
    z, _ = logits(6, 500, FP32, seed=3)
    u = torch.full((6,), 0.9)
    got = sample_tokens(z.to(cuda), u.to(cuda),
                        temperature=torch.tensor([-1.0, math.nan, 1.0, 1.0, 1.0, 1.0], device=cuda),
                        top_k=torch.tensor([0, 0, -3, 0, 0, 600], dtype=torch.int32, device=cuda),
                        top_p=torch.tensor([1.0, 1.0, 1.0, math.nan, 1.0, 7.0], device=cuda),
                        min_p=torch.tensor([0.0, 0.0, 0.0, 0.0, 9.0, 0.0], device=cuda))[0].cpu().tolist()
    rows = z.double().numpy()
    want = [ref.sample(r, 0.9)[0] for r in rows]
    want[0], want[1], want[4] = int(np.argmax(rows[0])), int(np.argmax(rows[1])), int(np.argmax(rows[4]))
    assert got == want


def test_more_rows_than_a_set_of_launches(cuda):
    """5000 rows with options of their own: the second set starts where the first ends."""
    print("sample 5000 rows", flush=True)
    b, v = 5000, 130
    z, u = logits(b, v, FP16, seed=9)
    g = torch.Generator().manual_seed(2)
    rand = lambda: torch.rand(b, generator=g)  # noqa: E731
    check(cuda, z, u, temperature=torch.where(rand() < 0.2, 0.0, 0.3 + rand()),
          top_k=torch.randint(0, v + 5, (b,), generator=g).int(), top_p=0.3 + 0.8 * rand(), min_p=0.1 * rand())
    check(cuda, z, u)
    check(cuda, z, u, min_p=0.2)


def test_endless_temperature_per_row(cuda):
    """A row's infinite temperature draws evenly from what is kept, a denormal one the maximum."""
    z = torch.randn(3, 20000, generator=torch.Generator().manual_seed(0))
    z[:, ::3] = -math.inf
    u = torch.full((3,), 0.6)
    for options in ({}, {"top_k": 100}, {"top_p": 0.5}, {"min_p": 0.2}, {"top_k": 9000, "top_p": 0.9}):
        check(cuda, z, u, temperature=torch.tensor([math.inf, 1e-40, 3e38]), **options)


@pytest.mark.parametrize("b", [4, 5])
def test_few_and_many_rows(cuda, b):
    """Either side of the rows for which the border is searched in a launch of its own: the same tokens."""
    z, u = logits(5, 60000, BF16, seed=21)
    options = {"top_k": 300, "top_p": 0.8, "temperature": 1.2}
    want = sample_tokens(z.to(cuda), u.to(cuda), **options)
    got = sample_tokens(z[:b].to(cuda), u[:b].to(cuda), **options)
    assert torch.equal(got[0], want[0][:b]) and torch.equal(got[1], want[1][:b])
    check(cuda, z[:b], u[:b], **options)


def test_two_calls_at_once(cuda):
    z, u = (t.to(cuda) for t in logits(40, 50257, BF16, seed=8))
    options = [{"top_p": 0.9}, {"top_k": 70, "temperature": 0.7}]
    want = [sample_tokens(z, u, **o) for o in options]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in range(5):
        for stream, o in zip(streams, options):
            with torch.cuda.stream(stream):
                got.append(sample_tokens(z, u, **o))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))


def test_frequencies(cuda):
    """Equally spaced random numbers draw every token as often as its probability says."""
    z = torch.randn(1, 300, generator=torch.Generator().manual_seed(0))
    n = 20000
    u = (torch.arange(n) + 0.5) / n
    tokens, logprobs = sample_tokens(z.to(cuda).expand(n, 300), u.to(cuda))
    p = torch.softmax(z[0].double(), 0)
    counts = torch.bincount(tokens.cpu(), minlength=300)
    assert (counts - n * p).abs().max() <= 1.01  # a token's interval holds its length's points, give or take one
    assert (logprobs.cpu() - p.log()[tokens.cpu()]).abs().max() <= 1e-5


@pytest.mark.parametrize("b", [1, 30])
def test_in_a_graph_and_on_another_stream(cuda, b):
    print(f"sample capture b={b}", flush=True)
    z, u = (t.to(cuda) for t in logits(b, 40000, BF16, seed=b))
    options = {"temperature": 0.9, "top_k": 3000, "top_p": 0.9, "min_p": 0.001}
    want = sample_tokens(z, u, **options)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = sample_tokens(z, u, **options)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(want, other))
    graphs, outs = [], []
    for _ in range(2):  # two graphs of one process
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(sample_tokens(z, u, **options))
    for step in range(4):
        u.copy_(torch.rand(b, generator=torch.Generator().manual_seed(step)))
        z.copy_(z.roll(step, 1))
        for graph in graphs:
            graph.replay()
        want = sample_tokens(z, u, **options)
        for out in outs:
            assert all(torch.equal(a, c) for a, c in zip(out, want))
        torch.cuda.synchronize()


@pytest.mark.parametrize("v, dtype, mode", [(151936, BF16, "none"), (151936, BF16, "all"), (151936, FP32, "top_p"),
                                            (1 << 21, BF16, "top_p"), (1 << 21, FP32, "none")])
def test_large_vocabularies(cuda, v, dtype, mode):
    print(f"sample v={v} {dtype} {mode}", flush=True)
    z, u = logits(2, v, dtype, seed=11)
    for i in range(2):
        assert ref.border_distance(z[i].double().numpy(), float(u[i]), **MODES[mode]) > 1e-11
    check(cuda, z, u, **MODES[mode])
