"""Whether a call may take the HIP kernels, and which path served each call.

The integration point of the reference's attention dispatch
(engine/streaming.py:355-373, :414-548) for this library:

* :func:`hip_attention_available` / :func:`hip_logprob_available` /
  :func:`hip_distill_available` / :func:`hip_embedding_available` /
  :func:`hip_sampling_available` / :func:`hip_paged_available` /
  :func:`hip_adjust_logits_available` answer for one call's tensors.  Under ``THUNDERSYNC_HIP=off`` (or ``auto`` without a
  loadable library) the answer is no; under ``require`` a library that cannot
  load raises at every call (``_lib.library``), and a loaded one is used
  without a trial, so that a kernel that cannot run on the device fails at
  the call instead of falling through; under ``auto`` the kernels are taken
  once a trial -- forward and backward of a tiny problem, once per
  ``(device, dtype, head_dim)`` -- has run on that device
  (:func:`thundersync_amd.capability.kernel_runs`).
* :func:`count_attention_path` / :func:`attention_path_counts` record, per
  path name, how many attention calls it served (the operators count
  ``hip`` per forward launch and ``hip_backward`` per backward launch).

The operators themselves never consult this module: they always run the
kernels and raise when they cannot; choosing another path is the caller's.
"""

from __future__ import annotations

import threading
from collections import Counter

import torch

from . import _lib
from .capability import kernel_runs

HIP_PATH = "hip"
HIP_BACKWARD_PATH = "hip_backward"

_counts: Counter[str] = Counter()
_counts_lock = threading.Lock()


def count_attention_path(name: str, calls: int = 1) -> None:
    """Record ``calls`` attention calls served by path ``name``."""
    with _counts_lock:
        _counts[name] += calls


def attention_path_counts() -> dict[str, int]:
    """Attention calls served per path in this process, cumulative, by name."""
    with _counts_lock:
        return dict(sorted(_counts.items()))


def reset_attention_path_counts() -> None:
    with _counts_lock:
        _counts.clear()


def attention_trial(device: torch.device, dtype: torch.dtype, head_dim: int) -> None:
    """Eight queries over a 16-key bottom-right window, 4 query heads on one KV
    head: the forward and every input gradient, finite."""
    from .attention import causal_attention

    g = torch.Generator(device=device).manual_seed(0)

    def leaf(*shape):
        return torch.randn(*shape, device=device, dtype=dtype, generator=g).requires_grad_()

    q, k, v = leaf(1, 4, 8, head_dim), leaf(16, 1, head_dim), leaf(16, 1, head_dim)
    out = causal_attention(q, [k], [v], head_dim ** -0.5)
    grads = torch.autograd.grad(out.float().square().sum(), (q, k, v))
    if not all(bool(t.isfinite().all()) for t in (out, *grads)):
        raise RuntimeError("HIP attention trial produced nonfinite values")


def logprob_trial(device: torch.device, dtype: torch.dtype, dim: int) -> None:
    """Five rows over a 300-token head: logprob, entropy and the hidden gradient, finite."""
    from .fused_logprob import fused_logprob_entropy

    g = torch.Generator(device=device).manual_seed(0)
    h = torch.randn(5, dim, device=device, dtype=dtype, generator=g).requires_grad_()
    w = torch.randn(300, dim, device=device, dtype=dtype, generator=g) * 0.02
    t = torch.randint(0, 300, (5,), device=device, generator=g)
    lp, ent = fused_logprob_entropy(h, w, t, chunk=4)
    (grad,) = torch.autograd.grad((lp + ent).sum(), (h,))
    if not all(bool(x.isfinite().all()) for x in (lp, ent, grad)):
        raise RuntimeError("HIP logprob trial produced nonfinite values")


def distill_trial(device: torch.device, dtype: torch.dtype, dim: int) -> None:
    """Five rows against four teacher logits each over a 300-token head: losses and the hidden gradient, finite."""
    from .fused_distill import fused_distill

    g = torch.Generator(device=device).manual_seed(0)
    h = torch.randn(5, dim, device=device, dtype=dtype, generator=g).requires_grad_()
    w = torch.randn(300, dim, device=device, dtype=dtype, generator=g) * 0.02
    ids = torch.randint(0, 300, (5, 4), device=device, generator=g)
    loss = fused_distill(h, w, ids, torch.randn(5, 4, device=device, generator=g), chunk=4)
    (grad,) = torch.autograd.grad(loss.sum(), (h,))
    if not all(bool(x.isfinite().all()) for x in (loss, grad)):
        raise RuntimeError("HIP distillation trial produced nonfinite values")


def embedding_trial(device: torch.device, dtype: torch.dtype, dim: int) -> None:
    """Forty tokens of a 30-row table: the rows themselves and as many gradients."""
    from .embedding import embedding

    g = torch.Generator(device=device).manual_seed(0)
    w = torch.randn(30, dim, device=device, dtype=dtype, generator=g).requires_grad_()
    ids = torch.randint(0, 30, (40,), device=device, generator=g)
    out = embedding(ids, w)
    (grad,) = torch.autograd.grad(out, w, torch.ones_like(out))
    if not bool((out == w[ids]).all()) or not bool((grad[:, 0] == torch.bincount(ids, minlength=30)).all()):
        raise RuntimeError("HIP embedding trial produced other rows or gradients")


def sampling_trial(device: torch.device, dtype: torch.dtype, vocab: int) -> None:
    """Two rows of one likely token each, drawn plainly and through every filter."""
    from .sampling import sample_tokens

    z = torch.zeros(2, vocab, device=device, dtype=dtype)
    z[0, 0] = z[1, vocab - 1] = 60.0
    u = torch.full((2,), 0.5, device=device)
    for options in ({}, {"temperature": 0.7, "top_k": 2, "top_p": 0.9, "min_p": 0.1}):
        if sample_tokens(z, u, **options)[0].tolist() != [0, vocab - 1]:
            raise RuntimeError("HIP sampling trial drew other tokens")


def paged_trial(device: torch.device, dtype: torch.dtype, row: int) -> None:
    """A token of two KV heads stored in caches of 8 and 16 bits, and the attention that sees it alone: its value."""
    from .paged import PagedCache, append_tokens, paged_attention

    ones = torch.ones(1, 2, row, device=device, dtype=dtype)
    batch = (torch.zeros(1, 1, device=device, dtype=torch.int32), torch.ones(1, device=device, dtype=torch.int32))
    for bits in (8, 16):
        cache = PagedCache.empty(1, 16, 2, row, dtype=dtype, bits=bits, device=device)
        append_tokens(cache, *batch, ones, 3 * ones)
        if not bool((paged_attention(ones, cache, *batch, 1.0) == 3).all()):
            raise RuntimeError("HIP paged attention trial read another value")


def adjust_logits_trial(device: torch.device, dtype: torch.dtype, vocab: int) -> None:
    """One row: a penalty on its first token, a bias on the same, nothing allowed but it."""
    from .logits import adjust_logits

    token = torch.zeros(1, 1, device=device, dtype=torch.int64)
    allowed = torch.zeros(1, (vocab + 31) // 32, device=device, dtype=torch.int32)
    allowed[0, 0] = 1
    z = adjust_logits(torch.full((1, vocab), 4.0, device=device, dtype=dtype), history=token, repetition=2.0,
                      presence=1.0, bias_ids=token, bias=token.float() + 3.0, allowed=allowed)
    if float(z[0, 0]) != 4.0 or not bool((z[0, 1:] == -torch.inf).all()):
        raise RuntimeError("HIP logits trial gave other values")


def _available(like: torch.Tensor, kernel: str, key: int, trial,
               dtypes=(torch.bfloat16, torch.float16)) -> bool:
    if not like.is_cuda or like.dtype not in dtypes:
        return False
    if _lib.library() is None:  # off, or auto without a library; require raises
        return False
    if _lib.resolved_setting() == "require":
        return True
    return kernel_runs(kernel, like, key, trial)


def hip_attention_available(query: torch.Tensor) -> bool:
    """Whether this query (any layout with the head dim last) may take the HIP attention."""
    from .attention import kernel_head_dim

    if kernel_head_dim(int(query.shape[-1])) is None:
        return False
    return _available(query, "hip_attention", int(query.shape[-1]), attention_trial)


def hip_logprob_available(hidden: torch.Tensor) -> bool:
    """Whether these hidden states may take the HIP fused logprob (bf16 and
    fp16 on MFMA; fp32 and fp64 at their own precision)."""
    return _available(hidden, "hip_logprob", int(hidden.shape[-1]), logprob_trial,
                      (torch.bfloat16, torch.float16, torch.float32, torch.float64))


def hip_distill_available(hidden: torch.Tensor) -> bool:
    """Whether these hidden states may take the HIP distillation (the fused logprob's types)."""
    return _available(hidden, "hip_distill", int(hidden.shape[-1]), distill_trial,
                      (torch.bfloat16, torch.float16, torch.float32, torch.float64))


def hip_embedding_available(weight: torch.Tensor) -> bool:
    """Whether this table may take the HIP embedding (bf16, fp16 and fp32)."""
    return _available(weight, "hip_embedding", int(weight.shape[-1]), embedding_trial,
                      (torch.bfloat16, torch.float16, torch.float32))


def hip_sampling_available(logits: torch.Tensor) -> bool:
    """Whether these logits may take the HIP sampling (bf16, fp16 and fp32)."""
    return _available(logits, "hip_sampling", int(logits.shape[-1]), sampling_trial,
                      (torch.bfloat16, torch.float16, torch.float32))


def hip_paged_available(query: torch.Tensor) -> bool:
    """Whether this query ``[tokens, heads, head_dim]`` may take the HIP paged cache and its attention (bf16 and fp16,
    head dims up to 256 that are multiples of eight)."""
    from .paged import stored_row

    if query.shape[-1] % 8 or not 8 <= query.shape[-1] <= 256:
        return False
    row = stored_row(int(query.shape[-1]))
    return _available(query, "hip_paged", row, paged_trial)


def hip_adjust_logits_available(logits: torch.Tensor) -> bool:
    """Whether these logits may take the HIP adjustment (bf16, fp16 and fp32)."""
    return _available(logits, "hip_adjust_logits", int(logits.shape[-1]), adjust_logits_trial,
                      (torch.bfloat16, torch.float16, torch.float32))
