"""Oracle of the adjustment of logits (CPU, fp64): one row at a time, from the definition."""

from __future__ import annotations

import math

import torch


def adjust(z, history=(), prompt=0, repetition=1.0, frequency=0.0, presence=0.0, bias_ids=(), bias=(), allowed=None):
    """The adjusted row: `history` a list of ids, `allowed` a list of truth values or None."""
    z = [float(x) for x in z]
    v = len(z)
    history = [int(t) for t in history]
    repetition = repetition if repetition > 0 else 1.0
    frequency = 0.0 if math.isnan(frequency) else frequency
    presence = 0.0 if math.isnan(presence) else presence
    for t in set(history):
        if 0 <= t < v:
            z[t] = z[t] / repetition if z[t] > 0 else z[t] * repetition
    made = history[max(prompt, 0):]
    for t in set(made):
        if 0 <= t < v:
            z[t] -= frequency * made.count(t) + presence
    for t, add in zip(bias_ids, bias):
        if 0 <= t < v:
            z[t] += float(add)
    if allowed is not None:
        z = [x if a else -math.inf for x, a in zip(z, allowed)]
    return torch.tensor(z, dtype=torch.float64)


def bound(z, want, frequency, presence, counts, bias_size, dtype):
    """Half a step of the result, and what fp32 loses of the terms on the way (each of a handful of roundings, half of 2^-23)."""
    size = z.double().abs() * 2 + abs(frequency) * counts + abs(presence) + bias_size
    return want.abs() * torch.finfo(dtype).eps / 2 + (size + want.abs()) * 8 * 2.0 ** -24 + torch.finfo(dtype).tiny
