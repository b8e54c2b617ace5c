"""Distillation from a teacher's top logits through the head, on the gfx950 kernels.

The companion of :mod:`thundersync_amd.fused_logprob` for on-policy
distillation: instead of the logprob of one target per row,
:func:`fused_distill` takes the K tokens and logits that a teacher returned
for each row and gives the row's divergence from the teacher,

    p = softmax over the row's teacher logits / temperature
    q = softmax over the whole vocabulary of (hidden . weight^T) / temperature
    loss = sum_k p_k (log p_k - log q_k)

without a ``[N, V]`` block of logits.  Gradients reach ``hidden`` always and
``weight`` when it requires one; the teacher's logits are data.

Slots with a negative token id or a logit of ``-inf`` are absent, so rows may
bring fewer than K; slots that name one token twice add up.  A row without
any present slot has loss 0 and no gradient, whatever its hidden state holds.
A token id at or past the vocabulary makes the row's loss NaN (and takes no
part in its gradient), as a target of the fused logprob does;
``THUNDERSYNC_CHECK_TARGETS=1`` checks the ids first and raises.

Forward: ``ts_distill_teacher`` turns the slots into probabilities and
``ts_distill_fwd`` takes the logits' log-sum-exp tile by tile on MFMA and the
logits at the slots.  Backward, per block of rows as in the fused logprob:
``ts_distill_dlogits`` recomputes the logits and writes
``grad / temperature (q - p)`` in the element type; the products with the
weight and the hidden states are the fused logprob's
(:func:`~thundersync_amd.fused_logprob.head_vjp`).  In fp16 an entry of that
block below 6e-8 is lost, so scale the loss as fp16 training does.

bf16 or fp16 (fp32 losses), fp32 or fp64 (losses of their own type, computed
at that precision).  GPU only: other dtypes and CPU tensors raise.
"""

from __future__ import annotations

import math
import os

import torch

from . import _lib
from .fused_logprob import (
    CHECK_TARGETS_ENV,
    ELEMENT_DTYPES,
    EXACT_DTYPES,
    _check_targets,
    _pad_dim,
    _rows_ok,
    _unit_stride,
    head_vjp,
    head_vjp_exact,
)
from .operator_profiling import device_role, operator_range

MAX_TOP = 1024  # teacher slots per row
TEACHER_DTYPES = (torch.bfloat16, torch.float16, torch.float32, torch.float64)


def _validate(hidden, weight, ids, logits, temperature):
    if hidden.dim() != 2:
        raise ValueError(f"hidden must be [N, D], got {tuple(hidden.shape)}")
    if weight.dim() != 2 or weight.shape[1] != hidden.shape[1]:
        raise ValueError(f"weight {tuple(weight.shape)} does not match hidden dim {hidden.shape[1]}")
    if ids.dim() != 2 or ids.shape[0] != hidden.shape[0]:
        raise ValueError(f"teacher_ids must be [N, K] with one row per hidden row, got {tuple(ids.shape)}")
    if logits.shape != ids.shape:
        raise ValueError(f"teacher_logits {tuple(logits.shape)} must have the shape of teacher_ids {tuple(ids.shape)}")
    if not 1 <= ids.shape[1] <= MAX_TOP:
        raise ValueError(f"1 to {MAX_TOP} teacher logits per row, got {ids.shape[1]}")
    if weight.shape[0] < 1 or hidden.shape[1] < 1:
        raise ValueError(f"an empty head: weight {tuple(weight.shape)}")
    if not (isinstance(temperature, (int, float)) and 0 < temperature < math.inf):
        raise ValueError(f"temperature must be a positive number, got {temperature!r}")
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"teacher_ids must be int64 or int32, got {ids.dtype}")
    if logits.dtype not in TEACHER_DTYPES:
        raise TypeError(f"teacher_logits must be bf16, fp16, fp32 or fp64, got {logits.dtype}")
    if not all(t.is_cuda for t in (hidden, weight, ids, logits)):
        raise RuntimeError("thundersync_amd fused distillation runs on the GPU only; got a CPU tensor")
    if any(t.device != hidden.device for t in (weight, ids, logits)):
        raise ValueError("hidden, weight, teacher_ids and teacher_logits must be on one device")
    if hidden.dtype not in ELEMENT_DTYPES + EXACT_DTYPES or weight.dtype != hidden.dtype:
        raise TypeError(
            "thundersync_amd fused distillation takes bf16, fp16, fp32 or fp64 hidden and weight of one dtype, got "
            f"{hidden.dtype}/{weight.dtype}"
        )
    if os.environ.get(CHECK_TARGETS_ENV, "0") not in ("", "0") and ids.numel():
        _check_targets(ids.amax(dim=1).clamp(min=0), weight.shape[0])  # an absent slot's negative id is no bad target


def _teacher(ids, logits, vocab, temperature, dtype):
    """(slot tokens, slot probabilities, row states) of a teacher's logits, for ``dtype``'s kernels."""
    lib = _lib.require_library()
    ids = ids.to(torch.int64).contiguous()
    logits = logits if logits.stride(1) == 1 and logits.stride(0) >= logits.shape[1] else logits.contiguous()
    n, k = ids.shape
    pitch = min((k + 3) // 4 * 4, MAX_TOP)
    slot_id = torch.empty(n, pitch, dtype=torch.int32, device=ids.device)
    slot_p = torch.empty(n, pitch, dtype=dtype, device=ids.device)
    state = torch.empty(n, dtype=torch.int32, device=ids.device)
    _lib.check(
        lib.ts_distill_teacher(ids.data_ptr(), logits.data_ptr(), logits.stride(0), _lib.dtype_code(logits.dtype), n, k,
                               vocab, float(temperature), slot_id.data_ptr(), slot_p.data_ptr(), pitch,
                               state.data_ptr(), _lib.dtype_code(dtype), _lib.stream_of(ids)),
        f"ts_distill_teacher(rows={n}, top={k}, vocab={vocab})",
    )
    return slot_id, slot_p, state


def _live_rows(h, state, scale):
    """``scale h`` with zeros in the rows without a teacher."""
    out = torch.empty(h.shape, dtype=h.dtype, device=h.device)
    _lib.check(
        _lib.require_library().ts_distill_rows(h.data_ptr(), max(h.stride(0), h.shape[1]), state.data_ptr(), h.shape[0],
                                               h.shape[1], float(scale), out.data_ptr(), h.shape[1],
                                               _lib.dtype_code(h.dtype), _lib.stream_of(h)),
        f"ts_distill_rows(rows={h.shape[0]}, dim={h.shape[1]})",
    )
    return out


def _forward(hidden, weight, ids, logits, temperature):
    lib = _lib.require_library()
    exact = hidden.dtype in EXACT_DTYPES
    dt = hidden.dtype if exact else torch.float32
    n, v, k = hidden.shape[0], weight.shape[0], ids.shape[1]
    slot_id, slot_p, state = _teacher(ids, logits, v, temperature, dt)
    slot_z = torch.empty_like(slot_p)
    pitch = slot_p.shape[1]
    loss = torch.empty(n, dtype=dt, device=hidden.device)
    lse = torch.empty(n, dtype=dt, device=hidden.device)
    code, stream = _lib.dtype_code(hidden.dtype), _lib.stream_of(hidden)
    if exact:
        # the logits over the temperature: of the rows divided by it
        h, w = _live_rows(_unit_stride(hidden), state, 1.0 / temperature), _unit_stride(weight)
        d = h.shape[1]
        ldw = max(w.stride(0), d)
        target = torch.zeros(n, dtype=torch.int64, device=h.device)
        unused = torch.empty(n, dtype=dt, device=h.device)
        ws_bytes = int(lib.ts_logprob_fwd_exact_workspace(n, v, code))
        ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=h.device)
        _lib.check(
            lib.ts_logprob_fwd_exact(h.data_ptr(), d, w.data_ptr(), ldw, target.data_ptr(), n, d, v, unused.data_ptr(),
                                     None, lse.data_ptr(), ws.data_ptr(), ws_bytes, code, stream),
            f"ts_logprob_fwd_exact(rows={n}, dim={d}, vocab={v})",
        )
        _lib.check(
            lib.ts_distill_scores(h.data_ptr(), d, w.data_ptr(), ldw, slot_id.data_ptr(), pitch, n, k, d,
                                  slot_z.data_ptr(), code, stream),
            f"ts_distill_scores(rows={n}, top={k}, dim={d})",
        )
        _lib.check(
            lib.ts_distill_loss(slot_id.data_ptr(), slot_p.data_ptr(), slot_z.data_ptr(), pitch, k, state.data_ptr(),
                                lse.data_ptr(), n, loss.data_ptr(), code, stream),
            f"ts_distill_loss(rows={n}, top={k})",
        )
    else:
        h, w = _rows_ok(_pad_dim(hidden)), _rows_ok(_pad_dim(weight))
        d = h.shape[1]
        ws_bytes = int(lib.ts_distill_fwd_workspace(n, v))
        ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=h.device)
        _lib.check(
            lib.ts_distill_fwd(h.data_ptr(), h.stride(0), w.data_ptr(), w.stride(0), n, d, v, float(temperature),
                               slot_id.data_ptr(), slot_p.data_ptr(), slot_z.data_ptr(), pitch, k, state.data_ptr(),
                               loss.data_ptr(), lse.data_ptr(), ws.data_ptr(), ws_bytes, code, stream),
            f"ts_distill_fwd(rows={n}, dim={d}, vocab={v}, top={k})",
        )
    return loss, lse, slot_id, slot_p, slot_z, state


def _backward(hidden, weight, lse, slot_id, slot_p, slot_z, state, grad, top, temperature, chunk, needs_weight_grad):
    lib = _lib.require_library()
    v, pitch = weight.shape[0], slot_p.shape[1]
    g = grad.to(lse.dtype).contiguous()
    code, stream = _lib.dtype_code(hidden.dtype), _lib.stream_of(hidden)
    slots = (slot_id, slot_p, slot_z)
    if hidden.dtype in EXACT_DTYPES:
        rows_in, w = _unit_stride(hidden), _unit_stride(weight)
        h = _live_rows(rows_in, state, 1.0 / temperature)
        h_weight = _live_rows(rows_in, state, 1.0) if needs_weight_grad else None
        d = h.shape[1]
        ldw = max(w.stride(0), d)
        none = torch.full((h.shape[0],), -1, dtype=torch.int64, device=h.device)
        # the logprob's coefficient kernel gives -q g; a row without a teacher has none
        coef = torch.where(state == 0, 0.0, g * (-1.0 / temperature))

        def dlogits(i, rows, dl, ld):
            _lib.check(
                lib.ts_logprob_dlogits_exact(h[i:].data_ptr(), d, w.data_ptr(), ldw, none[i:].data_ptr(),
                                             lse[i:].data_ptr(), None, coef[i:].data_ptr(), None, rows, d, v,
                                             dl.data_ptr(), ld, code, stream),
                f"ts_logprob_dlogits_exact(rows={rows}, dim={d}, vocab={v})",
            )
            _lib.check(
                lib.ts_distill_slots(*(s[i:].data_ptr() for s in slots), pitch, top, lse[i:].data_ptr(),
                                     g[i:].data_ptr(), rows, 1.0, 1.0 / temperature, dl.data_ptr(), ld, code, stream),
                f"ts_distill_slots(rows={rows}, top={top})",
            )

        return head_vjp_exact(h, w, chunk, needs_weight_grad, dlogits, h_weight)
    h, w = _rows_ok(_pad_dim(hidden)), _rows_ok(_pad_dim(weight))
    # 0 x NaN is NaN in the weight gradient's product: rows without a teacher enter it as zeros
    h_weight = _live_rows(h, state, 1.0) if needs_weight_grad else None
    d = h.shape[1]

    def dlogits(i, rows, dl, ld):
        _lib.check(
            lib.ts_distill_dlogits(h[i:].data_ptr(), h.stride(0), w.data_ptr(), w.stride(0), rows, d, v,
                                   float(temperature), *(s[i:].data_ptr() for s in slots), pitch, top,
                                   state[i:].data_ptr(), lse[i:].data_ptr(), g[i:].data_ptr(), dl.data_ptr(), ld, code,
                                   stream),
            f"ts_distill_dlogits(rows={rows}, dim={d}, vocab={v}, top={top})",
        )

    return head_vjp(h, w, hidden.shape[1], chunk, needs_weight_grad, dlogits, h_weight)


class _FusedDistill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, ids, logits, temperature, chunk, needs_weight_grad):
        with torch.cuda.device(hidden.device), operator_range(
                "fused_distill_forward", role=device_role(hidden.device), tokens=hidden.shape[0],
                hidden=hidden.shape[1], vocab=weight.shape[0], top=ids.shape[1], dtype=hidden.dtype):
            loss, *saved = _forward(hidden, weight, ids, logits, temperature)
        ctx.save_for_backward(hidden, weight, *saved)
        ctx.top, ctx.temperature, ctx.chunk, ctx.needs_weight_grad = ids.shape[1], temperature, chunk, needs_weight_grad
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        hidden, weight, *saved = ctx.saved_tensors
        with torch.cuda.device(hidden.device), operator_range(
                "fused_distill_backward", role=device_role(hidden.device), tokens=hidden.shape[0],
                hidden=hidden.shape[1], vocab=weight.shape[0], weight_grad=ctx.needs_weight_grad):
            gh, gw = _backward(hidden, weight, *saved, grad, ctx.top, ctx.temperature, ctx.chunk,
                               ctx.needs_weight_grad)
        return gh, gw, None, None, None, None, None


def fused_distill(hidden: torch.Tensor, weight: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
                  *, temperature: float = 1.0, chunk: int = 1024) -> torch.Tensor:
    """Per-row KL(teacher's top tokens || student) without materialising ``[N, V]``: ``[N]``.

    ``hidden`` ``[N, D]``, ``weight`` ``[V, D]``, ``teacher_ids`` (int64 or
    int32) and ``teacher_logits`` ``[N, K]``, K up to 1024.  Both softmaxes are
    taken at ``temperature``; the loss is not multiplied by its square.
    """
    _validate(hidden, weight, teacher_ids, teacher_logits, temperature)
    return _FusedDistill.apply(hidden, weight, teacher_ids, teacher_logits, float(temperature), chunk,
                               weight.requires_grad)
