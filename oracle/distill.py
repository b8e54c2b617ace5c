"""Distillation oracle (CPU, fp64): KL(teacher's top tokens || student) per row and its gradients.

From the definition: p is the softmax over a row's present slots (token id of 0 or more, logit above -inf) of
teacher / T, slots of one token added together; q the softmax over the vocabulary of hidden . weight^T / T;
loss = sum p (log p - log q); dz = grad / T (q - p); dh = dz W, dW = dz^T h.  A row without a present slot has
loss 0 and gradient 0; one with an id past the vocabulary has loss NaN, and that slot no part in its gradient.

:func:`bounds` gives, per element, how far a computation in a narrower type may be off: see there.

Pinned by (tests/test_oracle_vocabulary.py): autograd of the composed torch expression, and central differences.
"""

from __future__ import annotations

import math

import torch


def teacher_probs(ids, teacher, vocab, temperature):
    """(p [N, V] fp64, present rows [N], rows with an id past the vocabulary [N])."""
    n = ids.shape[0]
    there = (ids >= 0) & (teacher != -math.inf)
    x = torch.where(there, teacher.double() / temperature, -math.inf)
    some = there.any(dim=1)
    slots = torch.where(some[:, None], torch.softmax(torch.where(some[:, None], x, 0.0), dim=1), 0.0)
    slots = torch.where(there, slots, 0.0)
    inside = there & (ids < vocab)
    p = torch.zeros(n, vocab, dtype=torch.float64)
    p.index_put_((torch.arange(n)[:, None].expand_as(ids)[inside], ids.long()[inside]), slots[inside], accumulate=True)
    return p, some, (there & (ids >= vocab)).any(dim=1)


def distill(hidden, weight, ids, teacher, grad, temperature=1.0):
    """{"loss", "dh", "dw", "p", "q", "z"} in fp64; rows without a teacher are taken as zeros."""
    p, some, bad = teacher_probs(ids, teacher, weight.shape[0], temperature)
    h, w = torch.where(some[:, None], hidden.double(), 0.0), weight.double()
    z = h @ w.T / temperature
    log_q = torch.log_softmax(z, dim=1)
    q = log_q.exp()
    loss = (torch.special.xlogy(p, p) - torch.where(p > 0, p * log_q, 0.0)).sum(dim=1)
    loss = torch.where(bad, math.nan, torch.where(some, loss, 0.0))
    g = torch.where(some, grad.double(), 0.0) / temperature
    dz = g[:, None] * (q - p)
    return {"loss": loss, "dh": dz @ w, "dw": dz.T @ h, "p": p, "q": q, "z": z, "g": g, "h": h, "w": w}


def bounds(ref, dtype, top, temperature=1.0):
    """How far loss, dh and dw may be off ``ref`` (an oracle's result), per element.

    With a = 2^-24 (fp32 sums; 2^-53 for fp64) and u the element type's half step:
    * a logit over T, in fp32 or fp64, is off by at most e = (D + 4) a max_v sum_d |h w| / T (D products added in any
      order).  bf16 and fp16: MFMA adds 16 products at a time, so the sum is rounded D / 16 + 20 times (the last of a
      block of its own), each time by a of what it then is: no more than sum_d |h w|, and of terms of either sign within
      |z| + 4 (sum_d (h w)^2)^(1/2), four deviations of its random walk;
    * its exponential by e + 4 ulp of the argument and the function, |z| <= Z: rel = e + (8 + 2 Z) a.  The sum of V of
      them is added in blocks, by at most a a step: 128 of a tile's 256 in a lane and 6 across the lanes, then
      V / 16384 tiles of a slot and 18 slots, three roundings each (fp32 and fp64: V / 512 of a thread and 16 across
      them); lse likewise;
    * the loss, a sum of K terms p (log p - z + lse), by 2 rel + (K + 8) a (its terms' size).
    * dz's entries are rounded to the element type twice at most (the exponential, its product with the row's
      factors) on top of that: each by (2 u + 2 rel + V a) g (q + p), and below the smallest normal number by
      2^-25 absolute (fp16);
    * their products' sums add (V + 2) a (N + 2) and the result's own rounding u.
    """
    a = 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24
    u = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}.get(dtype, a)
    h, w, g, p, q, z = (ref[k] for k in ("h", "w", "g", "p", "q", "z"))
    n, v = p.shape
    d = h.shape[1]
    finite = torch.isfinite(z)
    size = torch.where(finite, z.abs(), 0.0).amax(dim=1, keepdim=True) if v else z
    added = h.abs() @ w.abs().T
    if dtype in (torch.bfloat16, torch.float16):
        walk = torch.where(finite, z.abs() * temperature, math.inf) + 4 * ((h * h) @ (w * w).T).sqrt()
        added, steps, depth = torch.minimum(added, walk), d / 16 + 20, 134 + 3 * (v / 16384 + 18)
    else:
        steps, depth = d + 4, v / 512 + 16
    rel = steps * a * added.amax(dim=1, keepdim=True) / temperature + (8 + 2 * size) * a + depth * a
    terms = torch.where(p > 0, p * (torch.log(torch.where(p > 0, p, 1.0)).abs() + size + math.log(v) + 1), 0.0).sum(dim=1)
    loss = 2 * rel[:, 0] + (top + 8) * a * (1 + terms)
    tiny = 2.0 ** -24 if dtype == torch.float16 else 0.0
    dz = (2 * u + 2 * rel) * g.abs()[:, None] * (q + p) + tiny * (1 + g.abs()[:, None])
    grow = lambda x, count: x * (1 + (count + 2) * a)  # noqa: E731
    dh = grow(dz @ w.abs(), v) + (v + 2) * a * ((g.abs()[:, None] * (q + p)) @ w.abs()) + u * ref["dh"].abs() + tiny
    dw = grow(dz.T @ h.abs(), n) + (n + 2) * a * ((g.abs()[:, None] * (q + p)).T @ h.abs()) + u * ref["dw"].abs() + tiny
    return {"loss": loss, "dh": dh, "dw": dw}
