"""Sampling oracle (CPU, numpy, fp64): one row at a time, by sorting.

From the definition: weights w = exp((z - max z) / T) in the order of falling logit, equal ones by rising index;
the first k; of those, the ones whose predecessors weigh less than p times all of those; of those, w >= min_p;
always the first.  The token is the first in index order whose running sum of kept weights exceeds u times their
total; logprob = log(w / total).  T = 0: the first maximum.  A row with a NaN or nothing above -inf: (-1, NaN).

Pinned by tests/test_oracle_vocabulary.py (frequencies against the softmax, hand-worked rows).
"""

from __future__ import annotations

import math

import numpy as np


def kept(z, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(indices kept, rising; all weights)."""
    z = np.asarray(z, dtype=np.float64)
    top = z.max()
    with np.errstate(invalid="ignore"):
        w = np.where(z == top, 1.0, np.where(z == -math.inf, 0.0, np.exp((z - top) / temperature)))
    order = np.argsort(-z, kind="stable")
    order = order[z[order] > -math.inf]
    if 0 < top_k < len(order):
        order = order[:top_k]
    if top_p < 1:
        before = np.concatenate([[0.0], np.cumsum(w[order])[:-1]])
        n = int(np.count_nonzero(before < top_p * w[order].sum()))
        order = order[: max(n, 1)]
    first = order[0]
    order = order[w[order] >= min(min_p, 1.0)]
    return np.sort(order if len(order) else np.array([first])), w


def sample(z, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, logprob) of one row."""
    z = np.asarray(z, dtype=np.float64)
    if np.isnan(z).any() or z.max() == -math.inf:
        return -1, math.nan
    if not temperature > 0:
        return int(np.argmax(z)), 0.0
    chosen, w = kept(z, temperature, top_k, top_p, min_p)
    running = np.cumsum(w[chosen])
    at = int(np.searchsorted(running, u * running[-1], side="right"))
    if at >= len(chosen):
        at = int(np.flatnonzero(w[chosen] > 0)[-1])
    with np.errstate(divide="ignore"):
        return int(chosen[at]), float(np.log(w[chosen[at]] / running[-1]))


def border_distance(z, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """How near u * total is to a step of the running sum, relative to the total: a draw nearer than the rounding of
    64-bit sums (about V * 2^-53) could go either way."""
    chosen, w = kept(z, temperature, top_k, top_p, min_p)
    running = np.cumsum(w[chosen])
    return float(np.abs(running / running[-1] - u).min())
