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
``THUNDERSYNC_CHECK_TARGETS=1`` checks the present slots' ids first and raises.

A block of rows (:func:`~thundersync_amd.fused_logprob.backward_block_rows` of
``chunk``) has its ``[rows, V]`` block in the element type, one at a time (two
in a backward whose block was kept):

* no gradient: the tiles' statistics alone, for all rows;
* a frozen weight: the forward goes on, block by block, from the stored
  exponentials to ``q - p`` and its product with the weight, ``[N, D]`` in
  fp32, which the backward multiplies by the upstream gradient (no block
  outlives the call, and 2 N V D flops of logits formed again are saved).
  The block's 16-bit entries are rounded once, with the exponent range of a
  row's own reference, and the teacher's tokens are added in fp32;
* a trainable weight and one block of rows: the backward, which has the
  upstream gradient, wants the block that the forward stored.  It is kept where
  the blocks of all losses that wait for their backward then hold no more
  than ``KEPT_BYTES``; otherwise the backward stores it again, by the same
  kernels and with the same bits (:class:`_KeptBlocks`).  Its 16-bit entries
  are rounded twice, as exponentials and with the row's factor: 2 bytes of
  memory an entry, where the logits that would be rounded once take 4;
* a trainable weight and more rows: the backward forms the logits again, block
  by block, as the fused logprob does.

The products with the weight and the hidden states are the fused logprob's
(:func:`~thundersync_amd.fused_logprob.head_vjp`).  In fp16 an entry of the
block below 6e-8 is lost, so scale the loss of a trainable head as fp16
training does.

bf16 or fp16 (fp32 losses), fp32 or fp64 (losses of their own type, computed
at that precision).  GPU only: other dtypes and CPU tensors raise.
"""

from __future__ import annotations

import copy
import math
import os
import threading
import weakref

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
    backward_block_rows,
    head_vjp,
    head_vjp_exact,
)
from .operator_profiling import device_role, operator_range

MAX_TOP = 1024  # teacher slots per row
# Below it a logit over T, in fp32 octaves, has no digits left behind the point, and its exponential overflows
MIN_TEMPERATURE = 1e-6
# Blocks that wait for their backward, on a device: 2048 rows of a 16-bit vocabulary of 262144
KEPT_BYTES = 1 << 30
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
    if not (isinstance(temperature, (int, float)) and MIN_TEMPERATURE <= temperature < math.inf):
        raise ValueError(f"temperature must be a positive number of {MIN_TEMPERATURE} or more, got {temperature!r}")
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
        present = (ids >= 0) & (logits != -math.inf)  # an absent slot's id is no target
        _check_targets(torch.where(present, ids, 0).amax(dim=1), weight.shape[0])


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
        lib.ts_distill_teacher(ids.data_ptr(), logits.data_ptr(), max(logits.stride(0), k),  # one row: any stride
                               _lib.dtype_code(logits.dtype), n, k, vocab, float(temperature), slot_id.data_ptr(),
                               slot_p.data_ptr(), pitch, state.data_ptr(), _lib.dtype_code(dtype),
                               _lib.stream_of(ids)),
        f"ts_distill_teacher(rows={n}, top={k}, vocab={vocab})",
    )
    return slot_id, slot_p, state


def _live_rows(h, state):
    """``h`` with zeros in the rows without a teacher: 0 x NaN is NaN in the weight gradient's product."""
    out = torch.empty(h.shape, dtype=h.dtype, device=h.device)
    _lib.check(
        _lib.require_library().ts_distill_rows(h.data_ptr(), max(h.stride(0), h.shape[1]), state.data_ptr(), h.shape[0],
                                               h.shape[1], out.data_ptr(), _lib.dtype_code(h.dtype), _lib.stream_of(h)),
        f"ts_distill_rows(rows={h.shape[0]}, dim={h.shape[1]})",
    )
    return out


class _KeptBlocks:
    """The blocks that losses on a device keep until their backward, so that together they hold no more than
    ``KEPT_BYTES`` (a batch scored in sixteen calls of 2000 rows of 151936 would keep 9.7 GB).  Kept, a step of
    1999 rows of D 2048 takes 3.85 ms; stored again in the backward 5.07."""

    def __init__(self):
        self._lock, self._alive = threading.Lock(), []

    def take(self, rows, ld, like):
        """An empty ``[rows, ld]`` block like ``like``, or None where it would take the blocks past their bound."""
        with self._lock:
            self._alive = [r for r in self._alive if r() is not None]
            held = sum(t.nbytes for t in (r() for r in self._alive) if t is not None and t.device == like.device)
            if held + rows * ld * like.element_size() > KEPT_BYTES:
                return None
            block = torch.empty(rows, ld, dtype=like.dtype, device=like.device)
            self._alive.append(weakref.ref(block))  # lives as long as what autograd saves
            return block


_kept = _KeptBlocks()


class _Rows:
    """A call's tensors as its kernels take them, and what the kernels find out about each row."""

    def __init__(self, hidden, weight, ids, logits, temperature):
        self.exact = hidden.dtype in EXACT_DTYPES
        self.dtype = hidden.dtype if self.exact else torch.float32  # of losses and statistics
        self.top, self.temperature = ids.shape[1], float(temperature)
        self._operands(hidden, weight)
        self.slot_id, self.slot_p, self.state = _teacher(ids, logits, weight.shape[0], temperature, self.dtype)
        self.slot_z = torch.empty_like(self.slot_p)
        self.lse, self.loss = (torch.empty(self.n, dtype=self.dtype, device=hidden.device) for _ in range(2))
        self.row_scale = None

    def _operands(self, hidden, weight):
        self.d_in = hidden.shape[1]
        if self.exact:
            self.h, self.w = _unit_stride(hidden), _unit_stride(weight)
            self.ld = (weight.shape[0] + 3) // 4 * 4  # rows of whole 16-byte vectors
        else:
            self.h, self.w = (_rows_ok(_pad_dim(t)) for t in (hidden, weight))
            self.ld = (weight.shape[0] + 7) // 8 * 8
        self.n, self.d = self.h.shape
        self.v = weight.shape[0]
        self.ldh, self.ldw = max(self.h.stride(0), self.d), max(self.w.stride(0), self.d)
        self.code = _lib.dtype_code(hidden.dtype)

    def saved(self):
        return self.slot_id, self.slot_p, self.slot_z, self.state, self.lse

    @classmethod
    def again(cls, hidden, weight, saved, top, temperature):
        """The rows of a forward that saved ``saved``, in its backward."""
        rows = cls.__new__(cls)
        rows.exact, rows.top, rows.temperature = hidden.dtype in EXACT_DTYPES, top, temperature
        rows._operands(hidden, weight)
        rows.slot_id, rows.slot_p, rows.slot_z, rows.state, rows.lse = saved
        rows.dtype, rows.row_scale = rows.lse.dtype, None
        return rows

    def slots(self, i):
        pitch = self.slot_p.shape[1]
        return (self.slot_id[i:].data_ptr(), self.slot_p[i:].data_ptr(), self.slot_z[i:].data_ptr(), pitch, self.top,
                self.state[i:].data_ptr())

    def row(self, i):
        return self.h.data_ptr() + i * self.ldh * self.h.element_size()

    def what(self, name, rows):
        return lambda: f"{name}(rows={rows}, dim={self.d}, vocab={self.v}, top={self.top})"

    def logits(self, i, rows, block):
        """fp32 / fp64: rows ``[i, i + rows)`` of hidden . weight^T into ``block``."""
        lib = _lib.require_library()
        ws_bytes = int(lib.ts_matmul_exact_workspace(rows, self.v, self.d, self.code))
        ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=block.device)
        _lib.check(
            lib.ts_matmul_exact_ws(self.row(i), self.ldh, 1, self.w.data_ptr(), 1, self.ldw, rows, self.v, self.d,
                                   block.data_ptr(), self.ld, 0, ws.data_ptr(), ws_bytes, self.code,
                                   _lib.stream_of(block)),
            self.what("ts_matmul_exact_ws", rows),
        )

    def forward(self, i, rows, block):
        """Losses of rows ``[i, i + rows)``; with a ``block`` also what :meth:`finish` and :meth:`softmax` read.
        Returns the tiles' references (16-bit types)."""
        lib, stream = _lib.require_library(), _lib.stream_of(self.h)
        if self.exact:
            self.logits(i, rows, block)
            _lib.check(
                lib.ts_distill_fwd_exact(block.data_ptr(), self.ld, rows, self.v, self.temperature, *self.slots(i),
                                         self.loss[i:].data_ptr(), self.lse[i:].data_ptr(), self.code, stream),
                self.what("ts_distill_fwd_exact", rows),
            )
            return None
        ws_bytes = int(lib.ts_distill_fwd_workspace(rows, self.v))
        ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=self.h.device)
        _lib.check(
            lib.ts_distill_fwd(self.row(i), self.ldh, self.w.data_ptr(), self.ldw, rows, self.d, self.v,
                               self.temperature, *self.slots(i), self.loss[i:].data_ptr(), self.lse[i:].data_ptr(),
                               _lib.ptr(block), self.ld, self.scale(i), ws.data_ptr(), ws_bytes, self.code, stream),
            self.what("ts_distill_fwd", rows),
        )
        return ws[: ws_bytes // 2]

    def stored_again(self, i, rows, block):
        """``block`` and its tiles' references as a :meth:`forward` that kept them left them (what autograd saved
        stays as it is)."""
        again = copy.copy(self)
        again.slot_z, again.lse, again.loss = (torch.empty_like(t) for t in (self.slot_z, self.lse, self.lse))
        return again.forward(i, rows, block)

    def scale(self, i):
        return None if self.row_scale is None else self.row_scale[i:].data_ptr()

    def softmax(self, i, rows, block, references):
        """16-bit types: ``block`` to the softmax over ``row_scale``, without the slots' tokens."""
        slot_id, _, _, pitch, top, state = self.slots(i)
        _lib.check(
            _lib.require_library().ts_distill_softmax(block.data_ptr(), self.ld, references.data_ptr(), self.scale(i),
                                                      rows, self.v, slot_id, pitch, top, state, self.code,
                                                      _lib.stream_of(block)),
            self.what("ts_distill_softmax", rows),
        )

    def add_slots(self, unit):
        """16-bit types: the products with the weight to those of ``q - p``."""
        *slots, _ = self.slots(0)
        _lib.check(
            _lib.require_library().ts_distill_slots(unit.data_ptr(), self.scale(0), self.w.data_ptr(), self.ldw, self.n,
                                                    self.d, self.temperature, *slots, self.lse.data_ptr(), self.code,
                                                    _lib.stream_of(unit)),
            self.what("ts_distill_slots", self.n),
        )

    def finish(self, i, rows, block, references, grad, out):
        """``block`` (as :meth:`forward` left it) to the logits' gradient ``out`` (which may be the block)."""
        _lib.check(
            _lib.require_library().ts_distill_finish(
                block.data_ptr(), self.ld, _lib.ptr(references), rows, self.v, self.temperature, *self.slots(i),
                self.lse[i:].data_ptr(), None if grad is None else grad[i:].data_ptr(), out.data_ptr(), self.ld,
                self.code, _lib.stream_of(out)),
            self.what("ts_distill_finish", rows),
        )

    def unit_gradient(self, i, rows, dl, out, ws):
        """``out`` rows ``[i, i + rows)`` = ``dl`` . weight, not rounded to the element type."""
        lib, stream = _lib.require_library(), _lib.stream_of(out)
        if self.exact:
            status = lib.ts_matmul_exact_ws(dl.data_ptr(), self.ld, 1, self.w.data_ptr(), self.ldw, 1, rows, self.d,
                                            self.v, out[i:].data_ptr(), self.d, 0, ws.data_ptr(), ws.numel(),
                                            self.code, stream)
        else:
            status = lib.ts_logprob_grad_hidden_f32(dl.data_ptr(), self.ld, self.w.data_ptr(), self.ldw, rows, self.d,
                                                    self.v, out[i:].data_ptr(), ws.data_ptr(), ws.numel(), self.code,
                                                    stream)
        _lib.check(status, self.what("distill gradient of hidden", rows))

    def unit_workspace(self, sizes):
        lib = _lib.require_library()
        need = (lambda r: lib.ts_matmul_exact_workspace(r, self.d, self.v, self.code)) if self.exact else (
            lambda r: lib.ts_logprob_grad_hidden_workspace(r, self.d, self.v))
        return torch.empty(max(16, *(int(need(r)) for r in sizes)), dtype=torch.uint8, device=self.h.device)


def _forward(rows: _Rows, chunk, need_hidden, need_weight):
    """The losses, and what the backward wants: nothing, the hidden states' unit gradient, or a kept block and its
    tiles' references."""
    n, dev = rows.n, rows.h.device
    block_rows = min(max(1, int(chunk)), max(n, 1)) if rows.exact else backward_block_rows(n, chunk)
    frozen = need_hidden and not need_weight
    if n == 0:
        return (torch.empty(0, rows.d, dtype=rows.dtype, device=dev),) if frozen else ()
    kept = _kept.take(n, rows.ld, rows.h) if need_weight and n <= block_rows else None
    if kept is None and not (rows.exact or frozen):
        rows.forward(0, n, None)
        return ()
    block = torch.empty(min(block_rows, n), rows.ld, dtype=rows.h.dtype, device=dev) if kept is None else kept
    unit = torch.empty(n, rows.d, dtype=rows.dtype, device=dev) if frozen else None
    ws = rows.unit_workspace({block_rows, n % block_rows or block_rows}) if frozen else None
    if frozen and not rows.exact:
        rows.row_scale = torch.empty(n, 2, dtype=torch.float32, device=dev)
    references = None
    for i in range(0, n, block_rows):
        size = min(block_rows, n - i)
        references = rows.forward(i, size, block)
        if frozen:
            with operator_range("distill_head_coefficient", role=device_role(dev), rows=size, vocab=rows.v):
                if rows.exact:
                    rows.finish(i, size, block, None, None, block)
                else:
                    rows.softmax(i, size, block, references)
            with operator_range("distill_head_hidden_vjp", role=device_role(dev), rows=size, hidden=rows.d, vocab=rows.v):
                rows.unit_gradient(i, size, block, unit, ws)
    if frozen:
        if not rows.exact:
            rows.add_slots(unit)
        return (unit,)
    return () if kept is None else (kept, references)


def _backward_frozen(unit, state, grad, temperature, dtype, d_in):
    n, d = unit.shape
    out = torch.empty(n, d, dtype=dtype, device=unit.device)
    _lib.check(
        _lib.require_library().ts_distill_scale(unit.data_ptr(), grad.to(unit.dtype).contiguous().data_ptr(),
                                                state.data_ptr(), n, d, temperature, out.data_ptr(),
                                                _lib.dtype_code(dtype), _lib.stream_of(unit)),
        f"ts_distill_scale(rows={n}, dim={d})",
    )
    return out if d == d_in else out[:, :d_in].contiguous()


def _backward_trainable(rows: _Rows, grad, chunk, block, references):
    g = grad.to(rows.dtype).contiguous()
    h_weight = _live_rows(rows.h, rows.state)
    lib = _lib.require_library()
    one = not rows.exact and rows.n <= backward_block_rows(rows.n, chunk)

    def dlogits(i, size, dl, ld):
        if block is not None:
            rows.finish(i, size, block, references, g, dl)
        elif rows.exact:
            rows.logits(i, size, dl)
            rows.finish(i, size, dl, None, g, dl)
        elif one:
            rows.finish(i, size, dl, rows.stored_again(i, size, dl), g, dl)
        else:
            _lib.check(
                lib.ts_distill_dlogits(rows.row(i), rows.ldh, rows.w.data_ptr(), rows.ldw, size, rows.d, rows.v,
                                       rows.temperature, *rows.slots(i), rows.lse[i:].data_ptr(), g[i:].data_ptr(),
                                       dl.data_ptr(), ld, rows.code, _lib.stream_of(dl)),
                rows.what("ts_distill_dlogits", size),
            )

    if rows.exact:
        return head_vjp_exact(rows.h, rows.w, chunk, True, dlogits, h_weight)
    return head_vjp(rows.h, rows.w, rows.d_in, chunk, True, dlogits, h_weight)


class _FusedDistill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, ids, logits, temperature, chunk, need_hidden, need_weight):
        with _lib.device_of(hidden), operator_range(
                "fused_distill_forward", role=device_role(hidden.device), tokens=hidden.shape[0],
                hidden=hidden.shape[1], vocab=weight.shape[0], top=ids.shape[1], dtype=hidden.dtype):
            rows = _Rows(hidden, weight, ids, logits, temperature)
            kept = _forward(rows, chunk, need_hidden, need_weight)
        ctx.frozen, ctx.chunk, ctx.top, ctx.temperature = not need_weight, chunk, rows.top, rows.temperature
        if need_weight:
            ctx.save_for_backward(hidden, weight, *rows.saved(), *kept)
        elif need_hidden:
            ctx.save_for_backward(*kept, rows.state)
            ctx.dtype, ctx.d_in, ctx.vocab = hidden.dtype, hidden.shape[1], weight.shape[0]
        return rows.loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        with _lib.device_of(grad), operator_range(
                "fused_distill_backward", role=device_role(grad.device), tokens=grad.shape[0],
                weight_grad=not ctx.frozen):
            if ctx.frozen:
                unit, state = ctx.saved_tensors
                gh, gw = _backward_frozen(unit, state, grad, ctx.temperature, ctx.dtype, ctx.d_in), None
            else:
                hidden, weight, *saved = ctx.saved_tensors
                block, references = [*saved[5:], None, None][:2]
                rows = _Rows.again(hidden, weight, saved[:5], ctx.top, ctx.temperature)
                gh, gw = _backward_trainable(rows, grad, ctx.chunk, block, references)
        return gh, gw, None, None, None, None, None, None


def fused_distill(hidden: torch.Tensor, weight: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
                  *, temperature: float = 1.0, chunk: int = 1024) -> torch.Tensor:
    """Per-row KL(teacher's top tokens || student) without materialising ``[N, V]``: ``[N]``.

    ``hidden`` ``[N, D]``, ``weight`` ``[V, D]``, ``teacher_ids`` (int64 or
    int32) and ``teacher_logits`` ``[N, K]``, K up to 1024.  Both softmaxes are
    taken at ``temperature`` (1e-6 or more); the loss is not multiplied by its square.
    """
    _validate(hidden, weight, teacher_ids, teacher_logits, temperature)
    grad = torch.is_grad_enabled()
    return _FusedDistill.apply(hidden, weight, teacher_ids, teacher_logits, float(temperature), chunk,
                               grad and hidden.requires_grad, grad and weight.requires_grad)
