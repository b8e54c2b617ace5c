"""Distillation through a trainable head: what losses that wait for their backward hold, and heads wide enough for
every token tile."""

from __future__ import annotations

import pytest
import torch

from thundersync_amd import fused_distill as module
from thundersync_amd.fused_distill import fused_distill

pytestmark = pytest.mark.gpu

BF16, FP16, FP32, FP64 = torch.bfloat16, torch.float16, torch.float32, torch.float64


def inputs(cuda, n, d, v, k, dtype, seed, wscale=0.05):
    g = torch.Generator(device=cuda).manual_seed(seed)
    h = torch.randn(n, d, generator=g, device=cuda).to(dtype).requires_grad_()
    w = (torch.randn(v, d, generator=g, device=cuda) * wscale).to(dtype).requires_grad_()
    ids = torch.randint(0, v, (n, k), generator=g, device=cuda)
    ids[:, 0] = v - 1  # the last token of the last tile
    teacher = torch.randn(n, k, generator=g, device=cuda) * 2
    return h, w, ids, teacher, torch.rand(n, generator=g, device=cuda) + 0.5


def exact(h, w, ids, teacher, grad):
    """(loss, dz, dh, dw) in fp64."""
    h, w, grad = h.detach().double(), w.detach().double(), grad.double()
    p = torch.zeros(h.shape[0], w.shape[0], dtype=FP64, device=h.device)
    p.scatter_add_(1, ids, torch.softmax(teacher.double(), dim=1))
    log_q = torch.log_softmax(h @ w.T, dim=1)
    dz = (log_q.exp() - p) * grad[:, None]
    return (torch.special.xlogy(p, p) - p * log_q).sum(dim=1), dz, dz @ w, dz.T @ h


@pytest.mark.parametrize("n, d, dtype", [
    (800, 64, BF16), (800, 64, FP16), (50, 64, BF16), (24, 64, FP16), (200, 64, FP32), (24, 64, FP32), (50, 64, FP64),
])
def test_losses_that_wait_for_their_backward(cuda, n, d, dtype, monkeypatch):
    """Together they keep blocks of no more than the bound (here the weight's size), and each has the same gradients,
    with a block kept (one of 50 rows, two of 24, none of more than 64) or without."""
    print(f"distill waiting losses n={n} d={d} {dtype}", flush=True)
    v, k, calls = 20011, 5, 6
    h, w, ids, teacher, grad = inputs(cuda, n, d, v, k, dtype, n)
    grad = grad.to(dtype if dtype == FP64 else torch.float32)
    want = torch.autograd.grad(fused_distill(h, w, ids, teacher), (h, w), grad)  # kept
    monkeypatch.setattr(module, "KEPT_BYTES", w.numel() * dtype.itemsize)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    losses = [fused_distill(h, w, ids, teacher) for _ in range(calls)]
    torch.cuda.synchronize()
    block, weight = n * v * dtype.itemsize, w.numel() * dtype.itemsize
    # per row: 8 places of slots (token, probability, logit), state, lse, loss; a block's tile statistics; memory comes
    # in pieces of 512 bytes
    rows = n * (8 * 20 + 24) + 8 * 512
    held = torch.cuda.memory_allocated() - before
    assert held <= calls * rows + 1.06 * weight, (held, rows, weight)
    assert (held >= block) == (block <= weight)
    torch.cuda.reset_peak_memory_stats()
    start = torch.cuda.memory_allocated()
    got = torch.autograd.grad(losses[-1], (h, w), grad)  # has kept nothing
    torch.cuda.synchronize()
    assert n < 800 or torch.cuda.max_memory_allocated() - start <= 1.5 * block
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    for loss in losses[:-1]:
        got = torch.autograd.grad(loss, (h, w), grad, retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        torch.autograd.grad(loss, (h, w), 2 * grad)
    held = torch.cuda.memory_allocated() - before
    del losses, loss
    fused_distill(h, w, ids, teacher)  # dropped without a backward
    waiting = fused_distill(h, w, ids, teacher)  # has the place again
    torch.cuda.synchronize()
    assert (torch.cuda.memory_allocated() - before >= block) == (block <= weight)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(waiting, (h, w), grad), want))


@pytest.mark.parametrize("n, d, dtype", [(300, 64, BF16), (48, 64, FP16), (600, 128, FP16), (2305, 64, BF16)])
def test_every_tile_of_a_wide_head(cuda, n, d, dtype):
    """Losses, dh row by row, dw by tiles of 256 tokens, over a whole vocabulary and every token tile (320 among them,
    2305 rows in several blocks).  Each of the three roundings (an exponential, a block's entry, the result) is off by u
    of its value at most, and errors of entries of either sign add as the entries do: 3 u of a row's or tile's root mean
    square; a tile left out is 1 of dw's and 4 % of dh's.  (The softmax's own entries: teachers name tokens whose row is
    zero.)  A loss: 2 (D / 16 + 20) 2^-24 sum |h w| <= 1e-5 of a logit and a slot's, a depth of 180 sums 2e-5, its own terms of at
    most 13 another 2e-5; the last, partial tile left out is 8e-4."""
    v, k = 151936, 7
    print(f"distill wide head n={n} d={d} {dtype}", flush=True)
    h, w, ids, teacher, grad = inputs(cuda, n, d, v, k, dtype, n)
    with torch.no_grad():
        w[:k] = 0
    ids = ids % k
    loss = fused_distill(h, w, ids, teacher)
    dh, dw = torch.autograd.grad(loss, (h, w), 256 * grad)  # fp16's smallest entries
    want, _, want_dh, want_dw = exact(h, w, ids, teacher, 256 * grad)
    u = torch.finfo(dtype).eps / 2
    assert (loss.double() - want).abs().max() <= 1e-4
    rms = lambda x: x.double().pow(2).mean(dim=-1).sqrt()  # noqa: E731
    assert (rms(dh.double() - want_dh) <= 3 * u * rms(want_dh)).all()
    last = (v - 1) // 256 * 256
    for got, ref in ((dw[256:last], want_dw[256:last]), (dw[last:], want_dw[last:]), (dw[:256], want_dw[:256])):
        rows = min(256, got.shape[0])
        assert (rms((got.double() - ref).reshape(-1, rows * d)) <= 3 * u * rms(ref.reshape(-1, rows * d))).all()
