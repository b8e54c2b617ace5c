"""Distillation through a frozen 16-bit head: the hidden states' gradient is as near as its own rounding lets it be,
and keeps small probabilities."""

from __future__ import annotations

import math

import pytest
import torch

from thundersync_amd.fused_distill import fused_distill

pytestmark = pytest.mark.gpu

BF16, FP16, FP64 = torch.bfloat16, torch.float16, torch.float64


def exact(h, w, ids, teacher, grad, temperature):
    """dh in fp64."""
    h, w = h.detach().double(), w.double()
    p = torch.zeros(h.shape[0], w.shape[0], dtype=FP64, device=h.device)
    p.scatter_add_(1, ids, torch.softmax(teacher.double() / temperature, dim=1))
    return ((torch.softmax(h @ w.T / temperature, dim=1) - p) * (grad.double() / temperature)[:, None]) @ w


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("n, d, v, k, temperature", [(48, 1024, 151936, 20, 1.0), (300, 512, 32003, 64, 2.0),
                                                     (7, 520, 4099, 1, 0.7), (20, 64, 5000, 300, 1.0)])
def test_the_error_is_the_results_rounding(cuda, n, d, v, k, temperature, dtype):
    """A teacher's few tokens are the gradient's largest terms: a block that rounds them has 1.4 times the error of the
    exact result's own rounding.  What is left is that rounding and the softmax's, whose entries' errors add over all the
    tokens: 1.15 covers those of these spreads (worked out in fp64) and the sampling."""
    print(f"distill frozen rounding n={n} d={d} v={v} k={k} T={temperature} {dtype}", flush=True)
    g = torch.Generator(device=cuda).manual_seed(n)
    h = torch.randn(n, d, generator=g, device=cuda).to(dtype).requires_grad_()
    w = (torch.randn(v, d, generator=g, device=cuda) * (1.5 / math.sqrt(d))).to(dtype)
    with torch.no_grad():
        top = ((h @ w.T).float() + torch.randn(n, v, generator=g, device=cuda)).topk(k, dim=1)
    teacher, ids = top.values + 3.0, top.indices
    grad = torch.rand(n, generator=g, device=cuda) + 0.5
    (dh,) = torch.autograd.grad(fused_distill(h, w, ids, teacher, temperature=temperature), h, grad)
    want = exact(h, w, ids, teacher, grad, temperature)
    error = lambda x: (x.double() - want).pow(2).mean().sqrt().item()  # noqa: E731
    assert error(dh) <= 1.15 * error(want.to(dtype)), (error(dh), error(want.to(dtype)))


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_small_probabilities_count(cuda, dtype):
    """Rows of equal logits over a whole vocabulary: the softmax's 6.6e-6 an entry is below fp16's normal numbers, and
    a block of it is off by 0.4 % everywhere, in one direction.  The head's rows have a mean, which the teacher's tokens
    cancel: that direction shows.  Bound: the result's rounding, and the fp32 sums over V of products of the mean's
    size, (V / 16) 2^-24 of them at most."""
    n, d, v, k = 33, 64, 151936, 7
    print(f"distill small probabilities {dtype}", flush=True)
    g = torch.Generator(device=cuda).manual_seed(0)
    w = (0.05 + 0.001 * torch.randn(v, d, generator=g, device=cuda)).to(dtype)
    h = torch.zeros(n, d, device=cuda, dtype=dtype, requires_grad=True)
    ids = torch.randint(0, v, (n, k), generator=g, device=cuda)
    teacher = torch.randn(n, k, generator=g, device=cuda)
    grad = torch.ones(n, device=cuda)
    (dh,) = torch.autograd.grad(fused_distill(h, w, ids, teacher), h, grad)
    want = exact(h, w, ids, teacher, grad, 1.0)
    bound = torch.finfo(dtype).eps / 2 * want.abs() + v / 16 * 2.0 ** -24 * 0.05 + 2.0 ** -25
    assert ((dh.double() - want).abs() <= bound).all(), ((dh.double() - want).abs() / bound).max().item()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("size", [1.0, 40.0, 90.0])
def test_gradients_stay_finite_at_the_lowest_temperature(cuda, size, dtype):
    """Logits over T of 9e7 step by 8 octaves in fp32 and so come to lie some octaves above their reference: the stored
    block has room for those."""
    g = torch.Generator(device=cuda).manual_seed(0)
    h = torch.randn(50, 64, generator=g, device=cuda)
    h = (h / h.norm(dim=1, keepdim=True)).to(dtype).requires_grad_()
    w = torch.randn(3000, 64, generator=g, device=cuda)
    w = (size * w / w.norm(dim=1, keepdim=True)).to(dtype)
    w[:50] = (size * h.detach()).to(dtype)  # a largest logit of `size` in every row
    ids = torch.randint(0, 3000, (50, 5), generator=g, device=cuda)
    loss = fused_distill(h, w, ids, torch.randn(50, 5, generator=g, device=cuda), temperature=1e-6)
    (dh,) = torch.autograd.grad(loss, h, torch.full_like(loss, 1e-6))
    assert loss.isfinite().all() and dh.isfinite().all()
