"""Sampling tokens from the head's logits with given random numbers, on the gfx950 kernel.

The rollout's counterpart of :mod:`thundersync_amd.fused_logprob`:
:func:`sample_tokens` draws one token per row of logits and gives its logprob
in the distribution it was drawn from (the behaviour policy of a policy
gradient), which for the default options is the model's own.

A row's weights are ``w = exp((logit - max) / temperature)``, ordered by
falling logit, equal logits by rising index.  Kept are

1. the first ``top_k`` (0: all),
2. of those, the ones whose predecessors weigh less than ``top_p`` times all
   of those (1 or more: all),
3. of those, the ones with ``w >= min_p`` (relative to the most likely token),

and always the first.  The token is the first in vocabulary order whose
running sum of kept weights exceeds ``uniform`` times their total, so a row's
token is a function of its logits, its options and its random number alone.
Sums are held in 64 bits: a running sum of 150,000 weights in 32 would move
tokens.  ``temperature`` 0 draws the first maximum.  A logit of ``-inf`` is
never drawn; a row with a NaN, or with nothing else than ``-inf``, gets token
-1 and logprob NaN.  GPU only: other dtypes and CPU tensors raise.
"""

from __future__ import annotations

import math

import torch

from . import _lib
from .operator_profiling import device_role, operator_range

DTYPES = (torch.bfloat16, torch.float16, torch.float32)
MAX_VOCAB = 1 << 21


def _per_row(name: str, value, logits: torch.Tensor, dtype: torch.dtype):
    """``(tensor or None, number)`` of an option given per row or once."""
    if not isinstance(value, torch.Tensor):
        if not isinstance(value, (int, float)) or math.isnan(value) or value < 0 or math.isinf(value):
            raise ValueError(f"{name} must be a finite number of 0 or more, got {value!r}")
        if dtype == torch.int32 and value != int(value):
            raise ValueError(f"{name} must be a whole number, got {value!r}")
        return None, value
    if value.shape != (logits.shape[0],):
        raise ValueError(f"{name} must be a number or one value per row ({logits.shape[0]}), got {tuple(value.shape)}")
    if value.dtype != dtype:
        raise TypeError(f"{name} per row must be {dtype}, got {value.dtype}")
    if value.device != logits.device:
        raise ValueError(f"{name} on {value.device} and logits on {logits.device}")
    return value.contiguous(), 0


def sample_tokens(logits: torch.Tensor, uniform: torch.Tensor, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """``(tokens int64 [B], logprobs fp32 [B])`` drawn from ``logits`` ``[B, V]``.

    ``uniform`` ``[B]`` (fp32 or fp64) holds a number in ``[0, 1)`` per row.
    ``temperature``, ``top_p`` and ``min_p`` are numbers or fp32 tensors
    ``[B]``, ``top_k`` a whole number or an int32 tensor ``[B]``; per-row values
    are not looked at on the host (a negative or NaN temperature counts as 0,
    a ``top_k`` below 1, a NaN ``top_p`` and a NaN ``min_p`` as none, a ``min_p``
    above 1 as 1).
    """
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"logits must be [B, V], got {tuple(logits.shape)}")
    if logits.shape[1] > MAX_VOCAB:
        raise ValueError(f"a vocabulary of at most {MAX_VOCAB}, got {logits.shape[1]}")
    if uniform.shape != (logits.shape[0],):
        raise ValueError(f"uniform must have one number per row ({logits.shape[0]}), got {tuple(uniform.shape)}")
    if logits.dtype not in DTYPES:
        raise TypeError(f"thundersync_amd sampling takes bf16, fp16 or fp32 logits, got {logits.dtype}")
    if uniform.dtype not in (torch.float32, torch.float64):
        raise TypeError(f"uniform must be fp32 or fp64, got {uniform.dtype}")
    options = [_per_row("temperature", temperature, logits, torch.float32),
               _per_row("top_k", top_k, logits, torch.int32),
               _per_row("top_p", top_p, logits, torch.float32),
               _per_row("min_p", min_p, logits, torch.float32)]
    if not logits.is_cuda or not uniform.is_cuda:
        raise RuntimeError("thundersync_amd sampling runs on the GPU only; got a CPU tensor")
    if uniform.device != logits.device:
        raise ValueError(f"uniform on {uniform.device} and logits on {logits.device}")
    lib = _lib.require_library()
    z = logits.detach()
    if z.shape[1] > 1 and z.stride(1) != 1:
        z = z.contiguous()
    u = uniform.contiguous()
    b, v = z.shape
    tokens = torch.empty(b, dtype=torch.int64, device=z.device)
    logprobs = torch.empty(b, dtype=torch.float32, device=z.device)
    (t_rows, t_all), (k_rows, k_all), (p_rows, p_all), (m_rows, m_all) = options
    filters = k_rows is not None or p_rows is not None or 1 < k_all < v or p_all < 1
    ws_bytes = int(lib.ts_sample_workspace(b, v, int(filters)))
    ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=z.device)
    with _lib.device_of(z), operator_range("sample_tokens", role=device_role(z.device), rows=b, vocab=v,
                                                     dtype=z.dtype):
        _lib.check(
            lib.ts_sample(z.data_ptr(), z.stride(0), b, v, u.data_ptr(), _lib.dtype_code(u.dtype), _lib.ptr(t_rows),
                          float(t_all), _lib.ptr(k_rows), min(int(k_all), MAX_VOCAB), _lib.ptr(p_rows), float(p_all),
                          _lib.ptr(m_rows), min(float(m_all), 1.0), tokens.data_ptr(), logprobs.data_ptr(),
                          ws.data_ptr(), ws_bytes, _lib.dtype_code(z.dtype), _lib.stream_of(z)),
            lambda: f"ts_sample(rows={b}, vocab={v}, {z.dtype})",
        )
    return tokens, logprobs
