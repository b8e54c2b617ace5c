"""Penalties, biases and grammar masks on logits, on the gfx950 kernel.

The step between the head and :func:`thundersync_amd.sampling.sample_tokens`.
For each row and token, in this order, in fp32 and rounded once:

1. ``z / repetition`` where z > 0, else ``z * repetition``, for tokens that
   occur in the row's history (its prompt and what it has generated);
2. ``- frequency * count - presence`` for tokens that occur ``count > 0`` times
   in the generated part;
3. ``+ bias``, the row's biases of the token summed in their order;
4. ``-inf`` for tokens that the row's mask does not allow.

A row whose mask allows nothing becomes all ``-inf``, for which the sampler draws
token -1.  No gradients or tangents, and GPU only: other dtypes and CPU tensors raise.
"""

from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from . import _lib
from .operator_profiling import device_role, operator_range
from .sampling import DTYPES, MAX_VOCAB

ID_DTYPES = (torch.int64, torch.int32)
MAX_BIASES = 1024


def _no_gradients(name: str, x: torch.Tensor):
    many = name == "logits"
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} require{'s'[many:]} grad, and adjust_logits has none: detach {'them' if many else 'it'}, or "
                           "call under torch.no_grad()")
    if forward_ad.unpack_dual(x).tangent is not None:
        raise RuntimeError(f"{name} {'have' if many else 'has'} a forward-mode tangent, and adjust_logits has none: detach "
                           f"{'them' if many else 'it'}")


def _penalty(name: str, value, logits: torch.Tensor):
    """``(tensor or None, number)`` of a penalty given per row or once."""
    if not isinstance(value, torch.Tensor):
        if not isinstance(value, (int, float)) or not abs(value) <= torch.finfo(torch.float32).max:
            raise ValueError(f"{name} must be a finite number (in fp32, as it is used), got {value!r}")
        if name == "repetition" and not torch.finfo(torch.float32).tiny <= value:
            raise ValueError(f"repetition must be above 0, got {value!r}")
        return None, float(value)
    _per_row(name, value, logits, (torch.float32,))
    _no_gradients(name, value)
    return value.contiguous(), 0.0


def _per_row(name: str, x: torch.Tensor, logits: torch.Tensor, dtypes, width: bool = False):
    if x.dim() != 1 + width or x.shape[0] != logits.shape[0]:
        raise ValueError(f"{name} must be [{logits.shape[0]}{', N' if width else ''}], a row each, got {tuple(x.shape)}")
    if x.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d).split('.')[1] for d in dtypes)}, got {x.dtype}")
    if x.device != logits.device:
        raise ValueError(f"{name} on {x.device} and logits on {logits.device}")


def _unit_rows(x: torch.Tensor) -> torch.Tensor:
    return x if x.shape[1] <= 1 or x.stride(1) == 1 else x.contiguous()


def _overlaps(out: torch.Tensor, logits: torch.Tensor) -> bool:
    """Whether the two share memory in another way than as the same rows."""
    if out.data_ptr() == logits.data_ptr() and all(n == 1 or s == t for n, s, t in zip(
            out.shape, out.stride(), logits.stride())):
        return False
    span = lambda x: (x.data_ptr(), x.data_ptr() + x.element_size() * (  # noqa: E731
        1 + sum((n - 1) * s for n, s in zip(x.shape, x.stride()))))
    (a, a_end), (b, b_end) = span(out), span(logits)
    return out.numel() > 0 and a < b_end and b < a_end


def pack_allowed(allowed: torch.Tensor) -> torch.Tensor:
    """The bits that ``allowed`` of :func:`adjust_logits` takes, ``[M, ceil(V / 32)]`` int32, of a bool mask ``[M, V]``."""
    if allowed.dim() != 2 or allowed.dtype != torch.bool:
        raise ValueError(f"a bool mask [M, V], got {allowed.dtype} {tuple(allowed.shape)}")
    # byte by byte of the words (of which the lowest comes first), a bit of all of them at a time
    bits = torch.nn.functional.pad(allowed, (0, -allowed.shape[1] % 32)).view(torch.uint8).unflatten(1, (-1, 8))
    packed = bits[..., 0].clone(memory_format=torch.contiguous_format)
    for i in range(1, 8):
        packed |= bits[..., i] << i
    return packed.view(torch.int32)


def adjust_logits(logits: torch.Tensor, *, history: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
                  prompt_lengths: torch.Tensor | None = None, repetition=1.0, frequency=0.0, presence=0.0,
                  bias_ids: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                  allowed: torch.Tensor | None = None, allowed_rows: torch.Tensor | None = None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """The adjusted ``logits`` ``[B, V]`` (fp32, bf16 or fp16), in ``out`` (which may be ``logits``) or a new tensor.

    ``history`` ``[B, H]`` (int64 or int32) holds each row's tokens, ``lengths``
    ``[B]`` (int32; None: H) how many, ``prompt_lengths`` ``[B]`` (int32; None: 0)
    how many of them were given and not generated.  ``repetition``,
    ``frequency`` and ``presence`` are numbers or fp32 tensors ``[B]``, whose
    values are not looked at on the host (a ``repetition`` not above 0 counts as 1, a
    NaN penalty as 0).  ``bias_ids`` (int64 or int32) and ``bias`` (fp32) ``[B,
    K]`` are sparse biases.  Ids outside ``[0, V)`` are passed over: padding.
    ``allowed`` ``[M, ceil(V / 32)]`` (int32) has bit ``v & 31`` of word ``v >>
    5`` set for an allowed token (:func:`pack_allowed`); row i has mask i, or
    ``allowed_rows`` ``[B]`` (int32) says which one, negative for none (one past
    them gives a row of NaN).
    """
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"logits must be [B, V], got {tuple(logits.shape)}")
    b, v = logits.shape
    if v > MAX_VOCAB:
        raise ValueError(f"a vocabulary of at most {MAX_VOCAB}, got {v}")
    if logits.dtype not in DTYPES:
        raise TypeError(f"thundersync_amd takes bf16, fp16 or fp32 logits, got {logits.dtype}")
    _no_gradients("logits", logits)
    penalties = [_penalty(*x, logits) for x in (("repetition", repetition), ("frequency", frequency),
                                                ("presence", presence))]
    if history is None:
        if lengths is not None or prompt_lengths is not None:
            raise ValueError("lengths and prompt_lengths are a history's")
        if any(t is not None or x != none for (t, x), none in zip(penalties, (1.0, 0.0, 0.0))):
            raise ValueError("penalties need a history")
    else:
        _per_row("history", history, logits, ID_DTYPES, width=True)
        for name, x in (("lengths", lengths), ("prompt_lengths", prompt_lengths)):
            if x is not None:
                _per_row(name, x, logits, (torch.int32,))
    if (bias_ids is None) != (bias is None):
        raise ValueError("bias_ids and bias go together")
    biases = 0
    if bias is not None:
        _per_row("bias_ids", bias_ids, logits, ID_DTYPES, width=True)
        _per_row("bias", bias, logits, (torch.float32,), width=True)
        _no_gradients("bias", bias)
        if bias.shape != bias_ids.shape or bias.shape[1] > MAX_BIASES:
            raise ValueError(f"bias must have the shape of bias_ids, of at most {MAX_BIASES} a row, got "
                             f"{tuple(bias.shape)} and {tuple(bias_ids.shape)}")
        biases = bias.shape[1]
    if allowed is not None:
        if allowed.dim() != 2 or allowed.shape[1] != (v + 31) // 32:
            raise ValueError(f"allowed must be [M, {(v + 31) // 32}], a bit for each of {v} tokens, got "
                             f"{tuple(allowed.shape)}")
        if allowed.dtype != torch.int32:
            raise TypeError(f"allowed must be int32, got {allowed.dtype}")
        if allowed.device != logits.device:
            raise ValueError(f"allowed on {allowed.device} and logits on {logits.device}")
        if allowed_rows is None and allowed.shape[0] != b:
            raise ValueError(f"a mask a row without allowed_rows: {allowed.shape[0]} masks for {b} rows")
    if allowed_rows is not None:
        if allowed is None:
            raise ValueError("allowed_rows without allowed")
        _per_row("allowed_rows", allowed_rows, logits, (torch.int32,))
    if out is not None and (out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device):
        raise ValueError(f"out must be like logits, {tuple(logits.shape)} {logits.dtype} on {logits.device}, got "
                         f"{tuple(out.shape)} {out.dtype} on {out.device}")
    if out is not None:
        _no_gradients("out", out)
    if out is not None and ((v > 1 and out.stride(1) != 1) or (b > 1 and out.stride(0) < v)):
        raise ValueError(f"out must have rows of their own, got strides {out.stride()}")
    if out is not None and _overlaps(out, logits):
        raise ValueError("out overlaps logits without being logits")
    if not logits.is_cuda:
        raise RuntimeError("thundersync_amd adjusts logits on the GPU only; got a CPU tensor")
    lib = _lib.require_library()
    z = _unit_rows(logits.detach())
    if out is None:
        out = torch.empty(b, v, dtype=z.dtype, device=z.device)
    ids = torch.int64
    if history is not None:
        ids, history = history.dtype, _unit_rows(history)
        lengths = None if lengths is None else lengths.contiguous()
        prompt_lengths = None if prompt_lengths is None else prompt_lengths.contiguous()
    if biases:
        ids = bias_ids.dtype if history is None else ids
        if bias_ids.dtype != ids:  # one type for both lists: an id outside the vocabulary stays outside in 32 bits
            bias_ids = bias_ids.clamp(-1, v).to(ids)
        bias_ids, bias = _unit_rows(bias_ids), _unit_rows(bias)
    if allowed is not None:
        allowed = _unit_rows(allowed)
        allowed_rows = None if allowed_rows is None else allowed_rows.contiguous()
    lead = lambda x: 0 if x is None else x.stride(0)  # noqa: E731
    (r_rows, r), (f_rows, f), (p_rows, p) = penalties
    with _lib.device_of(z), operator_range("adjust_logits", role=device_role(z.device), rows=b, vocab=v, dtype=z.dtype):
        _lib.check(
            lib.ts_adjust_logits(z.data_ptr(), z.stride(0), b, v, _lib.ptr(history), lead(history),
                                 0 if history is None else history.shape[1], _lib.ptr(lengths), _lib.ptr(prompt_lengths),
                                 _lib.ptr(r_rows), r, _lib.ptr(f_rows), f, _lib.ptr(p_rows), p, _lib.ptr(bias_ids),
                                 lead(bias_ids), _lib.ptr(bias), lead(bias), biases, _lib.ptr(allowed), lead(allowed),
                                 _lib.ptr(allowed_rows), 0 if allowed is None else allowed.shape[0],
                                 ids.itemsize, out.data_ptr(), max(out.stride(0), v), _lib.dtype_code(z.dtype),
                                 _lib.stream_of(z)),
            lambda: f"ts_adjust_logits(rows={b}, vocab={v}, {z.dtype})",
        )
    return out
