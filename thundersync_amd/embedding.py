"""Embedding lookup with a scale and its gradient by sorted tokens, on the gfx950 kernels.

:func:`embedding` is ``scale * weight[ids]`` for bf16, fp16 or fp32 tables
(one rounding of the fp32 product).  Its gradient with respect to the table is
dense, like ``torch.nn.functional.embedding``'s, but summed in fp32 in token
order without atomics (``ts_embedding_bwd`` sorts the positions by token), so
it has the same bytes every time, and rounded once.

A token id outside ``[0, vocab)`` gives a row of NaN and no gradient (a bad id
surfaces as a NaN loss, as a target of the fused logprob does);
``THUNDERSYNC_CHECK_TARGETS=1`` checks the ids first and raises.

:func:`use_hip_embedding` turns a model's ``torch.nn.Embedding`` modules into
:class:`HipEmbedding`, in place (a head tied to a table stays tied, hooks stay).
GPU only: other dtypes and CPU tensors raise in :func:`embedding`; the module
keeps torch's forward for them.
"""

from __future__ import annotations

import os

import torch
from torch.autograd import forward_ad

from . import _lib
from .fused_logprob import CHECK_TARGETS_ENV, _check_targets
from .operator_profiling import device_role, operator_range

DTYPES = (torch.bfloat16, torch.float16, torch.float32)
ID_DTYPES = (torch.int64, torch.int32)


def _on_one_device(ids, rows):
    if not ids.is_cuda or not rows.is_cuda:
        raise RuntimeError("thundersync_amd embedding runs on the GPU only; got a CPU tensor")
    if ids.device != rows.device:
        raise ValueError(f"ids on {ids.device} and rows on {rows.device}")


def _validate(ids, weight, scale, padding_idx):
    if weight.dim() != 2 or weight.shape[1] < 1:
        raise ValueError(f"weight must be [V, D], got {tuple(weight.shape)}")
    if ids.dtype not in ID_DTYPES:
        raise TypeError(f"ids must be int64 or int32, got {ids.dtype}")
    if not (isinstance(scale, (int, float)) and abs(scale) <= torch.finfo(torch.float32).max):
        raise ValueError(f"scale must be a finite number (in fp32, as it is used), got {scale!r}")
    if padding_idx is not None and not 0 <= padding_idx < weight.shape[0]:
        raise ValueError(f"padding_idx {padding_idx} is outside the vocabulary [0, {weight.shape[0]})")
    _on_one_device(ids, weight)
    if weight.dtype not in DTYPES:
        raise TypeError(f"thundersync_amd embedding takes a bf16, fp16 or fp32 weight, got {weight.dtype}")
    if os.environ.get(CHECK_TARGETS_ENV, "0") not in ("", "0"):
        _check_targets(ids.reshape(-1), weight.shape[0])


def _unit_rows(t: torch.Tensor) -> torch.Tensor:
    """``[N, D]`` with unit stride in the rows (which may repeat: a stride of 0)."""
    return t if t.shape[1] <= 1 or t.stride(1) == 1 else t.contiguous()


def embedding_forward(ids: torch.Tensor, weight: torch.Tensor, scale: float) -> torch.Tensor:
    """``scale * weight[ids]`` (ids of any shape), without autograd."""
    _on_one_device(ids, weight)
    lib = _lib.require_library()
    flat = ids.reshape(-1).to(torch.int64).contiguous()
    w = weight if weight.stride(1) == 1 and weight.stride(0) >= weight.shape[1] else weight.contiguous()
    v, d = w.shape
    out = torch.empty(*ids.shape, d, dtype=w.dtype, device=w.device)
    with _lib.device_of(w):
        _lib.check(
            lib.ts_embedding_fwd(flat.data_ptr(), flat.numel(), w.data_ptr(), max(w.stride(0), d), v, d, float(scale),
                                 out.data_ptr(), _lib.dtype_code(w.dtype), _lib.stream_of(w)),
            lambda: f"ts_embedding_fwd(tokens={flat.numel()}, vocab={v}, dim={d})",
        )
    return out


def embedding_backward(ids: torch.Tensor, grad_out: torch.Tensor, vocab: int, *, scale: float = 1.0,
                       padding_idx: int | None = None) -> torch.Tensor:
    """The table's gradient ``[vocab, D]`` for ``grad_out`` ``[*ids.shape, D]``."""
    _on_one_device(ids, grad_out)
    lib = _lib.require_library()
    d = grad_out.shape[-1]
    flat = ids.reshape(-1).to(torch.int64).contiguous()
    n = flat.numel()
    g = _unit_rows(grad_out.reshape(n, d))
    grad = torch.empty(vocab, d, dtype=g.dtype, device=g.device)
    ws_bytes = int(lib.ts_embedding_bwd_workspace(n, d))
    ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=g.device)
    with _lib.device_of(g):
        _lib.check(
            lib.ts_embedding_bwd(flat.data_ptr(), n, g.data_ptr(), g.stride(0), vocab, d,
                                 -1 if padding_idx is None else int(padding_idx), float(scale), grad.data_ptr(),
                                 ws.data_ptr(), ws_bytes, _lib.dtype_code(g.dtype), _lib.stream_of(g)),
            lambda: f"ts_embedding_bwd(tokens={n}, vocab={vocab}, dim={d})",
        )
    return grad


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.save_for_forward(ids)
        ctx.vocab, ctx.dtype, ctx.scale, ctx.padding_idx = weight.shape[0], weight.dtype, scale, padding_idx
        with operator_range(
                "embedding_forward", role=device_role(weight.device), tokens=ids.numel(), hidden=weight.shape[1],
                vocab=weight.shape[0], dtype=weight.dtype):
            return embedding_forward(ids, weight, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        (ids,) = ctx.saved_tensors
        with operator_range(
                "embedding_backward", role=device_role(grad.device), tokens=ids.numel(), hidden=grad.shape[-1],
                vocab=ctx.vocab):
            gw = embedding_backward(ids, grad.to(ctx.dtype), ctx.vocab, scale=ctx.scale, padding_idx=ctx.padding_idx)
        return None, gw, None, None

    @staticmethod
    def jvp(ctx, ids_tangent, weight_tangent, *_):
        (ids,) = ctx.saved_tensors
        return embedding_forward(ids, weight_tangent, ctx.scale)


def embedding(ids: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0,
              padding_idx: int | None = None) -> torch.Tensor:
    """``scale * weight[ids]``: ``[*ids.shape, D]`` for int64 or int32 ``ids`` of any shape.

    The row ``padding_idx`` of the table gets no gradient.  A table's forward-mode
    tangent reaches the rows.
    """
    _validate(ids, weight, scale, padding_idx)
    if not (weight.requires_grad and torch.is_grad_enabled()) and forward_ad.unpack_dual(weight).tangent is None:
        return embedding_forward(ids, weight.detach(), float(scale))
    return _Embedding.apply(ids, weight, float(scale), padding_idx)


class HipEmbedding(torch.nn.Embedding):
    """``torch.nn.Embedding`` on the HIP kernels; a call they do not serve (a CPU
    tensor, another dtype, the library switched off) runs torch's forward."""

    def forward(self, input):  # noqa: A002 - torch's name
        takes = (input.is_cuda and self.weight.is_cuda and input.dtype in ID_DTYPES and self.weight.dtype in DTYPES
                 and input.device == self.weight.device and self.embedding_dim > 0 and _lib.library() is not None)
        if not takes:
            return super().forward(input)
        return embedding(input, self.weight, padding_idx=self.padding_idx)


def use_hip_embedding(model: torch.nn.Module) -> int:
    """Make every plain ``torch.nn.Embedding`` below ``model`` a :class:`HipEmbedding`
    and return the count.  The modules stay the same objects, with their Parameter,
    hooks and attributes, under every name they go by.  Modules with ``max_norm``,
    ``scale_grad_by_freq`` or ``sparse`` and subclasses of their own are left alone."""
    count = 0
    for name, module in model.named_modules():
        if not name or type(module) is not torch.nn.Embedding:
            continue
        if module.max_norm is not None or module.scale_grad_by_freq or module.sparse:
            continue
        module.__class__ = HipEmbedding  # no state of its own
        count += 1
    return count
