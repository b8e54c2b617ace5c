"""Numbers that the kernels' fp32 cannot hold are refused; the smallest that it can are served."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import distill as ref
from thundersync_amd import embedding, fused_distill


@pytest.mark.parametrize("scale", [1e39, -1e300, math.inf, math.nan])
def test_embedding_scale(scale):
    with pytest.raises(ValueError, match="scale must be a finite number"):
        embedding.embedding(torch.zeros(3, dtype=torch.int64), torch.zeros(8, 4), scale=scale)


@pytest.mark.parametrize("temperature", [1e-300, 1e-38, 1e-7])
def test_distill_temperature(temperature):
    """z / T in fp32 octaves steps by more than an exponential's range: NaN losses."""
    with pytest.raises(ValueError, match="temperature must be a positive number of 1e-06 or more"):
        fused_distill.fused_distill(torch.zeros(4, 8), torch.zeros(16, 8), torch.zeros(4, 3, dtype=torch.int64),
                                    torch.zeros(4, 3), temperature=temperature)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("temperature", [1e-6, 1e-3])
def test_distill_at_low_temperatures(cuda, temperature, dtype):
    """Losses of 1e6 within the oracle's bound (an argument of that size), gradients finite."""
    print(f"distill T={temperature} {dtype}", flush=True)
    g = torch.Generator().manual_seed(0)
    h = torch.randn(9, 32, generator=g).to(dtype)
    w = (torch.randn(700, 32, generator=g) * 0.2).to(dtype)
    ids, teacher = torch.randint(0, 700, (9, 4), generator=g), torch.randn(9, 4, generator=g)
    want = ref.distill(h, w, ids, teacher, torch.ones(9), temperature)
    bound = ref.bounds(want, dtype, 4, temperature)["loss"]
    for train in (False, True):
        hc, wc = h.to(cuda).requires_grad_(), w.to(cuda).requires_grad_(train)
        loss = fused_distill.fused_distill(hc, wc, ids.to(cuda), teacher.to(cuda), temperature=temperature)
        grads = torch.autograd.grad(loss, [hc, wc] if train else hc, torch.full_like(loss, temperature))
        assert ((loss.double().cpu() - want["loss"]).abs() <= bound).all()
        assert all(x.isfinite().all() for x in grads)
