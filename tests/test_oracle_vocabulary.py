"""The oracles of distillation, embedding and sampling against something other than themselves (CPU)."""

from __future__ import annotations

import math

import numpy as np
import torch

from oracle import distill, embedding, sampling


def test_distill_against_autograd_and_differences():
    g = torch.Generator().manual_seed(0)
    n, d, v, k, t = 5, 7, 13, 4, 1.7
    h = torch.randn(n, d, generator=g, dtype=torch.float64, requires_grad=True)
    w = torch.randn(v, d, generator=g, dtype=torch.float64, requires_grad=True)
    ids = torch.randint(0, v, (n, k), generator=g)
    teacher = torch.randn(n, k, generator=g, dtype=torch.float64)
    ids[1, 2:] = -1
    teacher[2, 1:] = -math.inf
    ids[3] = -1
    ids[4, 1] = ids[4, 0]  # one token twice
    grad = torch.rand(n, generator=g, dtype=torch.float64) + 0.5
    ref = distill.distill(h.detach(), w.detach(), ids, teacher, grad, t)

    def loss_of(h, w):
        rows = []
        for i in range(n):
            slots = {}
            there = [j for j in range(k) if ids[i, j] >= 0 and teacher[i, j] > -math.inf]
            if not there:
                rows.append(torch.zeros((), dtype=torch.float64))
                continue
            p = torch.softmax(teacher[i, there] / t, dim=0)
            for j, x in zip(there, p):
                slots[int(ids[i, j])] = slots.get(int(ids[i, j]), 0) + x
            log_q = torch.log_softmax(h[i] @ w.T / t, dim=0)
            rows.append(sum(x * (torch.log(x) - log_q[tok]) for tok, x in slots.items()))
        return torch.stack(rows)

    loss = loss_of(h, w)
    assert torch.allclose(loss, ref["loss"], rtol=1e-12, atol=1e-12)
    dh, dw = torch.autograd.grad(loss, (h, w), grad)
    assert torch.allclose(dh, ref["dh"], rtol=1e-10, atol=1e-12)
    assert torch.allclose(dw, ref["dw"], rtol=1e-10, atol=1e-12)
    step = torch.randn(n, d, generator=g, dtype=torch.float64)
    with torch.no_grad():
        diff = ((loss_of(h + 1e-5 * step, w) - loss_of(h - 1e-5 * step, w)) * grad).sum() / 2e-5
    assert abs(diff - (ref["dh"] * step).sum()) < 1e-7


def test_distill_is_zero_where_student_and_teacher_agree():
    w = torch.eye(6, dtype=torch.float64)
    h = torch.randn(1, 6, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    ref = distill.distill(h, w, torch.arange(6)[None], h, torch.ones(1, dtype=torch.float64))
    assert ref["loss"].abs() < 1e-14 and ref["dh"].abs().max() < 1e-14


def test_embedding_against_torch():
    g = torch.Generator().manual_seed(2)
    w = torch.randn(9, 5, generator=g, requires_grad=True)
    ids = torch.randint(0, 9, (3, 4), generator=g)
    out = torch.nn.functional.embedding(ids, w, padding_idx=2)
    assert torch.equal(out, embedding.lookup(ids, w.detach()))
    grad = torch.randn(3, 4, 5, generator=g)
    (dw,) = torch.autograd.grad(out, w, grad)
    want = embedding.gradient(ids, grad, 9, padding_idx=2)
    assert ((dw - want).abs() <= embedding.gradient_bound(ids, grad, 9, padding_idx=2)).all()
    assert torch.isnan(embedding.lookup(torch.tensor([-1, 9]), w.detach())).all()


def test_sampling_frequencies_and_hand_worked_rows():
    z = np.log([0.1, 0.4, 0.3, 0.2])
    us = (np.arange(4000) + 0.5) / 4000
    tokens = [sampling.sample(z, u)[0] for u in us]
    assert np.allclose(np.bincount(tokens, minlength=4) / 4000, [0.1, 0.4, 0.3, 0.2], atol=1e-3)
    # the nucleus of 0.5: 0.4, then 0.3 (what is before it, 0.4, is below 0.5)
    assert set(sampling.sample(z, u, top_p=0.5)[0] for u in us) == {1, 2}
    assert abs(sampling.sample(z, 0.0, top_p=0.5)[1] - math.log(0.4 / 0.7)) < 1e-12
    assert sampling.sample(z, 0.99, top_k=2) == sampling.sample(z, 0.99, top_p=0.5)
    # top_p over what top_k keeps: of 0.4 and 0.3, 0.4 alone weighs 4/7 > 0.55
    assert sampling.sample(z, 0.99, top_k=2, top_p=0.55)[0] == 1
    assert sampling.sample(z, 0.99, min_p=0.7)[0] == 2
    # equal logits by index, greedy the first
    assert sampling.sample([1.0, 2.0, 2.0, 2.0], 0.99, top_k=2)[0] == 2
    assert sampling.sample([1.0, 2.0, 2.0], 0.99, temperature=0.0) == (1, 0.0)
    assert sampling.sample([-math.inf] * 3, 0.5)[0] == -1 and sampling.sample([0.0, math.nan], 0.5)[0] == -1
    assert sampling.sample([0.0, math.inf, 5.0, math.inf], 0.6) == (3, math.log(0.5))
