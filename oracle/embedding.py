"""Embedding oracle (CPU): the lookup in fp32 rounded once, the table's gradient in fp64.

``lookup`` is bit-exact: fp32(scale) * fp32(w), rounded to the table's type; NaN rows for ids outside the table.
``gradient`` is scale * the sum of grad_out's rows by id; ``gradient_bound`` is how far fp32 sums rounded once may
be off it: count - 1 additions and one product, each by 2^-24 of the sum of the absolute values, and the
result's half step.  Pinned by tests/test_oracle_vocabulary.py (torch's own embedding and its autograd).
"""

from __future__ import annotations

import math

import torch


def lookup(ids, weight, scale=1.0):
    ok = (ids >= 0) & (ids < weight.shape[0])
    rows = weight[torch.where(ok, ids, 0).long()].float() * torch.tensor(scale, dtype=torch.float32)
    return torch.where(ok[..., None], rows, math.nan).to(weight.dtype)


def _taken(ids, vocab, padding_idx):
    flat = ids.reshape(-1).long()
    keep = (flat >= 0) & (flat < vocab)
    return flat, keep if padding_idx is None else keep & (flat != padding_idx)


def gradient(ids, grad_out, vocab, scale=1.0, padding_idx=None):
    flat, keep = _taken(ids, vocab, padding_idx)
    rows = grad_out.reshape(flat.numel(), -1).double()
    return torch.zeros(vocab, rows.shape[1], dtype=torch.float64).index_add_(0, flat[keep], rows[keep]) * scale


def gradient_bound(ids, grad_out, vocab, scale=1.0, padding_idx=None):
    dtype = grad_out.dtype
    u = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}.get(dtype, 2.0 ** -24)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    sizes = gradient(ids, grad_out.abs(), vocab, abs(scale), padding_idx)
    flat, keep = _taken(ids, vocab, padding_idx)
    count = torch.bincount(flat[keep], minlength=vocab).double()[:, None]
    sums = (count + 1) * 2.0 ** -24 * sizes
    return sums + u * (gradient(ids, grad_out, vocab, scale, padding_idx).abs() + sums) + tiny
