"""A paged cache of keys and values, appending to it, and attention over it, on the gfx950 kernels.

The decoding step's side of :mod:`thundersync_amd.attention`: rollouts of every
length share one :class:`PagedCache`, whose pages of 16 to 256 tokens a page
table deals out to the sequences.

* :func:`append_tokens` puts new tokens' keys and values into their pages, and
  rotates query and key by position on the way;
* :func:`paged_attention` attends from a sequence's new tokens to all of its
  keys: one token a sequence, a few drafted ones, or a chunk of a prompt.

Both take the same description of a batch, read on the device, so that a
captured graph replays with new values: ``page_table`` ``[B, W]`` (int32 page
ids, a sequence's pages in order), ``lengths`` ``[B]`` (int32, tokens of each
sequence with the call's own; 0 for a row of padding) and ``offsets``
``[B + 1]`` (int32, the rows of the call that are each sequence's; None: one
each; rows before the first and behind the last are no sequence's, and zero in
what comes out).  A call's new tokens are the last of their sequence: token ``i`` of
``n`` has position ``length - n + i`` and sees the keys up to its own.

Held in 8 bits, keys and values are e4m3 codes times a scale for each 16 tokens
of a page and head.  Scales are powers of two, in an fp16 cache from 2^-15 on,
so that codes have no smaller steps than fp16: a value is ``code * scale``
exactly, in bf16 and fp16 too, attention over the codes is attention over those
values, and a block whose scale grows keeps its older codes' values (but for
bits that pass below e4m3's range).  The rounding to a code is the only one.

Bad input found on the device: a token past the page table, or whose page id is
no page of the cache, is stored nowhere, and attention rows that see such a key
are NaN; ``THUNDERSYNC_CHECK_TARGETS=1`` checks the batch first and raises.  A
block of 16 tokens that a call writes belongs to one sequence (sequences may
share pages that they only read).  There are no gradients and no tangents through a cache,
and no host path: other dtypes and CPU tensors raise.
"""

from __future__ import annotations

import ctypes
import math
import os

import torch
from torch.autograd import forward_ad

from . import _lib
from ._abi import PagedBatch, PagedCacheDesc
from .dispatch import count_attention_path
from .fused_logprob import CHECK_TARGETS_ENV
from .operator_profiling import device_role, operator_range

DTYPES = (torch.bfloat16, torch.float16)
CODES = torch.float8_e4m3fn
PAGE_SIZES = (16, 32, 64, 128, 256)
SCALE_TOKENS = 16  # tokens of a page that share a scale
ROWS = (64, 128, 192, 256)  # row lengths the kernels are built for
PATH = "hip_paged"  # the name under which attention_path_counts() has these calls


def stored_row(head_dim: int) -> int:
    """Elements of a stored row: the next length that the kernels take."""
    for row in ROWS:
        if 8 <= head_dim <= row and head_dim % 8 == 0:
            return row
    raise ValueError(f"head_dim must be a multiple of 8 from 8 to {ROWS[-1]}, got {head_dim}")


class PagedCache:
    """Pages ``[pages, kv_heads, page_size, row]`` of keys and of values.

    ``key`` and ``value`` are of ``dtype`` (16 bits) or ``torch.float8_e4m3fn``
    with fp32 ``key_scale`` and ``value_scale`` ``[pages, kv_heads, page_size //
    16]`` (8 bits).  Both are used in place; a page's ``[kv_heads, page_size,
    row]`` lies densely.  ``row`` is one of 64, 128, 192 and 256; a smaller
    ``head_dim`` (a multiple of 8) leaves zeros behind it, as :meth:`empty` does.
    The kernels are given what was checked here, so none of it can be set anew:
    other tensors are another cache.
    """

    _GIVEN = frozenset(("key", "value", "key_scale", "value_scale", "bits", "pages", "kv_heads", "page_size", "row",
                        "head_dim", "dtype"))

    def __init__(self, key: torch.Tensor, value: torch.Tensor, key_scale: torch.Tensor | None = None,
                 value_scale: torch.Tensor | None = None, *, dtype: torch.dtype | None = None,
                 head_dim: int | None = None):
        if key.dim() != 4 or key.shape != value.shape:
            raise ValueError(f"key and value must be [pages, kv_heads, page_size, row], got {tuple(key.shape)} and "
                             f"{tuple(value.shape)}")
        pages, heads, page_size, row = key.shape
        if row not in ROWS:
            raise ValueError(f"rows of {', '.join(map(str, ROWS))} elements, got {row}")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {', '.join(map(str, PAGE_SIZES))}, got {page_size}")
        if not 1 <= heads <= 1024 or pages < 1:
            raise ValueError(f"at least one page of 1 to 1024 heads, got {pages} of {heads}")
        head_dim = row if head_dim is None else head_dim
        if stored_row(head_dim) > row:
            raise ValueError(f"head_dim {head_dim} in rows of {row}")
        if key.dtype != value.dtype or key.dtype not in (*DTYPES, CODES):
            raise TypeError(f"key and value must both be bf16, fp16 or float8_e4m3fn, got {key.dtype} and {value.dtype}")
        self.bits = 8 if key.dtype == CODES else 16
        dtype = (torch.bfloat16 if self.bits == 8 else key.dtype) if dtype is None else dtype
        if dtype not in DTYPES or (self.bits == 16 and dtype != key.dtype):
            raise TypeError(f"a cache of {key.dtype} stands for bf16 or fp16 values, got {dtype}")
        scales = (pages, heads, page_size // SCALE_TOKENS)
        for name, scale, x in (("key_scale", key_scale, key), ("value_scale", value_scale, value)):
            if (scale is not None) != (self.bits == 8):
                raise ValueError(f"{name} goes with float8_e4m3fn pages, and only with them")
            if scale is not None:
                if scale.shape != scales or not scale.is_contiguous():
                    raise ValueError(f"{name} must be contiguous {scales}, got {tuple(scale.shape)}")
                if scale.dtype != torch.float32:
                    raise TypeError(f"{name} must be fp32, got {scale.dtype}")
                if scale.device != x.device:
                    raise ValueError(f"{name} on {scale.device} and pages on {x.device}")
        for x in (key, value):
            if x.requires_grad:
                raise ValueError("a cache holds no gradients")
            if x.stride()[1:] != (page_size * row, row, 1) or (pages > 1 and x.stride(0) < heads * page_size * row):
                raise ValueError(f"each page must be dense, got strides {x.stride()}")
            if x.data_ptr() % 16 or x.stride(0) % 16:
                raise ValueError("pages must begin at multiples of 16 bytes")
        if key.device != value.device:
            raise ValueError(f"key on {key.device} and value on {value.device}")
        self.key, self.value, self.key_scale, self.value_scale = key, value, key_scale, value_scale
        self.pages, self.kv_heads, self.page_size, self.row = pages, heads, page_size, row
        self.head_dim, self.dtype = head_dim, dtype
        stride = heads * page_size * row
        self._desc = PagedCacheDesc(
            key.data_ptr(), value.data_ptr(), _lib.ptr(key_scale), _lib.ptr(value_scale),
            key.stride(0) if pages > 1 else stride, value.stride(0) if pages > 1 else stride, pages, page_size, heads,
            head_dim, row, self.bits, _lib.dtype_code(dtype))
        self._ref = ctypes.byref(self._desc)

    def __setattr__(self, name, value):
        if name in self._GIVEN and "_ref" in self.__dict__:
            raise AttributeError(f"{name} of a PagedCache is what its kernels were given; make another over other tensors")
        super().__setattr__(name, value)

    @classmethod
    def empty(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, *, dtype: torch.dtype = torch.bfloat16,
              bits: int = 16, device="cuda") -> "PagedCache":
        """A cache of zeros."""
        if bits not in (8, 16):
            raise ValueError(f"bits must be 8 or 16, got {bits}")
        if dtype not in DTYPES:
            raise TypeError(f"a cache stands for bf16 or fp16 values, got {dtype}")
        shape = (pages, kv_heads, page_size, stored_row(head_dim))
        kv = [torch.zeros(shape, dtype=dtype if bits == 16 else CODES, device=device) for _ in range(2)]
        scales = [None, None] if bits == 16 else [
            torch.ones(pages, kv_heads, page_size // SCALE_TOKENS, device=device) for _ in range(2)]
        return cls(*kv, *scales, dtype=dtype, head_dim=head_dim)

    @property
    def device(self) -> torch.device:
        return self.key.device

    def values(self) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values ``[pages, kv_heads, page_size, head_dim]`` of ``dtype``: the
        pages themselves in 16 bits, new tensors of what the codes stand for in 8."""
        if self.bits == 16:
            return self.key[..., :self.head_dim], self.value[..., :self.head_dim]
        _on_the_gpu(self.key)
        lib = _lib.require_library()
        out = [torch.empty(self.pages, self.kv_heads, self.page_size, self.head_dim, dtype=self.dtype,
                           device=self.device) for _ in range(2)]
        with _lib.device_of(self.key), operator_range("paged_values", role=device_role(self.device), pages=self.pages):
            _lib.check(lib.ts_paged_values(self._ref, out[0].data_ptr(), out[1].data_ptr(), _lib.stream_of(self.key)),
                       lambda: f"ts_paged_values(pages={self.pages})")
        return out[0], out[1]


def rotary_table(positions: int, rotary_dim: int, *, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """``[positions, rotary_dim]`` fp32: cosines, then sines, of ``position *
    base ** (-2 j / rotary_dim)``.  The angles are formed in 64 bits: in 32 those
    of far positions are off by their rounding, 2^-24 of up to the position itself."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even, got {rotary_dim}")
    j = torch.arange(rotary_dim // 2, dtype=torch.float64, device=device)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * base ** (-2.0 / rotary_dim * j)
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def _on_the_gpu(*tensors):
    if not all(t.is_cuda for t in tensors):
        raise RuntimeError("thundersync_amd's paged cache runs on the GPU only; got a CPU tensor")


def _no_gradients(name: str, x: torch.Tensor):
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires grad, and there are no gradients through a paged cache: detach it, or call "
                           "under torch.no_grad()")
    if forward_ad.unpack_dual(x).tangent is not None:
        raise RuntimeError(f"{name} has a forward-mode tangent, and there are none through a paged cache: detach it")


def _rows(name: str, x: torch.Tensor, cache: PagedCache) -> torch.Tensor:
    """``x`` ``[T, heads, head_dim]`` with dense, 16-byte aligned rows."""
    if x.dim() != 3 or x.shape[2] != cache.head_dim:
        raise ValueError(f"{name} must be [T, heads, {cache.head_dim}], got {tuple(x.shape)}")
    if x.dtype != cache.dtype:
        raise TypeError(f"{name} must be {cache.dtype} as the cache, got {x.dtype}")
    _no_gradients(name, x)
    a, b, c = x.stride()
    if c == 1 and (a | b) % 8 == 0 and x.data_ptr() % 16 == 0:
        return x
    return x.detach().clone(memory_format=torch.contiguous_format)


def _batch(cache, page_table, lengths, offsets, tokens, like, writes=False) -> tuple[PagedBatch, list]:
    """The call's description, and what has to live until it has run."""
    if page_table.dim() != 2 or lengths.shape != (page_table.shape[0],):
        raise ValueError(f"page_table must be [B, W] and lengths [B], got {tuple(page_table.shape)} and "
                         f"{tuple(lengths.shape)}")
    b, w = page_table.shape
    if offsets is None:
        if tokens != b:
            raise ValueError(f"without offsets each sequence has one row: {tokens} rows for {b} sequences")
    elif offsets.shape != (b + 1,):
        raise ValueError(f"offsets must be [B + 1] = [{b + 1}], got {tuple(offsets.shape)}")
    device = like.device
    for name, x in (("page_table", page_table), ("lengths", lengths), ("offsets", offsets)):
        if x is None:
            continue
        if x.dtype != torch.int32:
            raise TypeError(f"{name} must be int32, got {x.dtype}")
        if x.device != device:
            raise ValueError(f"{name} on {x.device} and rows on {device}")
    if cache.device != device:
        raise ValueError(f"cache on {cache.device} and rows on {device}")
    _on_the_gpu(like)
    table = page_table if w <= 1 or page_table.stride(1) == 1 else page_table.contiguous()
    lengths = lengths.contiguous()
    offsets = None if offsets is None else offsets.contiguous()
    if os.environ.get(CHECK_TARGETS_ENV, "0") not in ("", "0"):
        _check_batch(cache, table, lengths, offsets, tokens, writes)
    return PagedBatch(table.data_ptr(), lengths.data_ptr(), _lib.ptr(offsets), table.stride(0), w, b), \
        [table, lengths, offsets]


def _check_batch(cache, table, lengths, offsets, tokens, writes):
    b, w = table.shape
    n = torch.ones_like(lengths) if offsets is None else offsets[1:] - offsets[:-1]
    if offsets is not None and (int(offsets[0]) < 0 or int(offsets[-1]) > tokens or bool((n < 0).any())):
        raise ValueError(f"offsets must be rising places among the {tokens} rows")
    bad = (lengths < 0) | (lengths > w * cache.page_size) | ((lengths > 0) & (lengths < n))
    used = torch.arange(w, device=table.device) < (lengths[:, None] + cache.page_size - 1) // cache.page_size
    bad |= (used & ((table < 0) | (table >= cache.pages))).any(dim=1)
    if bool(bad.any()):
        s = int(bad.nonzero()[0])
        raise ValueError(f"sequence {s} has {int(lengths[s])} tokens, {int(n[s])} of them new, over pages "
                         f"{table[s][used[s]].tolist()} of {cache.pages}")
    if writes and b:
        # the blocks of 16 tokens that each sequence writes
        per, w16 = cache.page_size // SCALE_TOKENS, w * cache.page_size // SCALE_TOKENS
        block = torch.arange(w16, device=table.device)
        first, last = (lengths - n).clamp(min=0) // SCALE_TOKENS, (lengths - 1) // SCALE_TOKENS
        written = (block >= first[:, None]) & (block <= last[:, None]) & (n > 0)[:, None]
        ids = (table.long().repeat_interleave(per, dim=1) * per + block % per)[written]
        if ids.unique().numel() != ids.numel():
            raise ValueError("two sequences write to one block of 16 tokens")


def append_tokens(cache: PagedCache, page_table: torch.Tensor, lengths: torch.Tensor, key: torch.Tensor,
                  value: torch.Tensor, *, query: torch.Tensor | None = None, offsets: torch.Tensor | None = None,
                  rotary: torch.Tensor | None = None, positions: torch.Tensor | None = None,
                  interleaved: bool = False) -> torch.Tensor | None:
    """Put ``key`` and ``value`` ``[T, kv_heads, head_dim]`` into the cache; the rotated ``query`` ``[T, heads, head_dim]``.

    With ``rotary`` ``[P, R]`` (see :func:`rotary_table`; R a multiple of 16) the
    first R elements of each query and key row are rotated by the row of the
    table at its position, or at ``positions`` ``[T]`` (int32): pairs are
    elements ``j`` and ``j + R / 2``, ``2 j`` and ``2 j + 1`` where
    ``interleaved``.  The rotation is computed in fp32 and rounded once, to the
    cache's form; a position outside the table gives NaN.  Query rows that are no sequence's are zero.
    """
    key, value = _rows("key", key, cache), _rows("value", value, cache)
    if key.shape != value.shape or key.shape[1] != cache.kv_heads:
        raise ValueError(f"key and value must be [T, {cache.kv_heads}, {cache.head_dim}], got {tuple(key.shape)} and "
                         f"{tuple(value.shape)}")
    t = key.shape[0]
    heads = 0
    if query is not None:
        query = _rows("query", query, cache)
        heads = query.shape[1]
        if query.shape[0] != t:
            raise ValueError(f"query has {query.shape[0]} rows and key {t}")
    r = 0
    if rotary is not None:
        if rotary.dim() != 2 or rotary.shape[1] % 16 or not 16 <= rotary.shape[1] <= cache.head_dim:
            raise ValueError(f"rotary must be [P, R] with R a multiple of 16 up to {cache.head_dim}, got "
                             f"{tuple(rotary.shape)}")
        if rotary.dtype != torch.float32:
            raise TypeError(f"rotary must be fp32, got {rotary.dtype}")
        _no_gradients("rotary", rotary)
        rotary = rotary.detach().contiguous()
        rotary = rotary if rotary.data_ptr() % 16 == 0 else rotary.clone()
        r = rotary.shape[1]
    if positions is not None:
        if positions.shape != (t,):
            raise ValueError(f"positions must be [T] = [{t}], got {tuple(positions.shape)}")
        if positions.dtype != torch.int32:
            raise TypeError(f"positions must be int32, got {positions.dtype}")
        positions = positions.contiguous()
    for name, x in (("query", query), ("value", value), ("rotary", rotary), ("positions", positions)):
        if x is not None and x.device != key.device:
            raise ValueError(f"{name} on {x.device} and key on {key.device}")
    batch, keep = _batch(cache, page_table, lengths, offsets, t, key, writes=True)
    lib = _lib.require_library()
    out = None if query is None else torch.empty(t, heads, cache.head_dim, dtype=cache.dtype, device=key.device)
    qs = (0, 0) if query is None else query.stride()[:2]
    with _lib.device_of(key), operator_range("append_tokens", role=device_role(key.device), tokens=t,
                                             heads=heads, kv_heads=cache.kv_heads, head_dim=cache.head_dim, bits=cache.bits):
        _lib.check(
            lib.ts_paged_append(cache._ref, ctypes.byref(batch), t, _lib.ptr(query), qs[0], qs[1], heads, _lib.ptr(out),
                                key.data_ptr(), key.stride(0), key.stride(1), value.data_ptr(), value.stride(0),
                                value.stride(1), _lib.ptr(rotary), 0 if rotary is None else rotary.shape[0], r,
                                int(interleaved), _lib.ptr(positions), _lib.stream_of(key)),
            lambda: f"ts_paged_append(tokens={t}, heads={heads}/{cache.kv_heads}, head_dim={cache.head_dim}, "
                    f"bits={cache.bits})",
        )
    del keep
    return out


def paged_attention(query: torch.Tensor, cache: PagedCache, page_table: torch.Tensor, lengths: torch.Tensor,
                    scale: float, *, offsets: torch.Tensor | None = None) -> torch.Tensor:
    """``softmax(scale q k) v`` of ``query`` ``[T, heads, head_dim]`` over the keys of its sequences, ``[T, heads, head_dim]``.

    Query head ``h`` reads KV head ``h // (heads // kv_heads)``.  Keys that a row does not see
    (those of tokens behind it, and what lies behind a sequence's end in its last
    page) have no part in it whatever they hold.  A row without keys is zero.  Scores, weights and sums
    are fp32; for the product with the values a weight is rounded to the query's type.  A call takes
    fewer than 2^24 rows (tokens times heads).
    """
    q = _rows("query", query, cache)
    t, heads, _ = q.shape
    if heads < 1 or heads % cache.kv_heads:
        raise ValueError(f"query heads {heads} are not a multiple of KV heads {cache.kv_heads}")
    if not isinstance(scale, (int, float)) or not math.isfinite(scale):
        raise ValueError(f"scale must be a finite number, got {scale!r}")
    batch, keep = _batch(cache, page_table, lengths, offsets, t, q)
    lib = _lib.require_library()
    out = torch.empty(t, heads, cache.head_dim, dtype=cache.dtype, device=q.device)
    ref = ctypes.byref(batch)
    with _lib.device_of(q), operator_range("paged_attention", role=device_role(q.device), tokens=t, heads=heads,
                                           kv_heads=cache.kv_heads, head_dim=cache.head_dim, bits=cache.bits):
        ws_bytes = int(lib.ts_paged_attention_workspace(cache._ref, ref, t, heads))
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device) if ws_bytes else None
        _lib.check(
            lib.ts_paged_attention(cache._ref, ref, t, q.data_ptr(), q.stride(0), q.stride(1), heads, float(scale),
                                   out.data_ptr(), _lib.ptr(ws), ws_bytes, _lib.stream_of(q)),
            lambda: f"ts_paged_attention(tokens={t}, heads={heads}/{cache.kv_heads}, head_dim={cache.head_dim}, "
                    f"bits={cache.bits})",
        )
    count_attention_path(PATH)
    del keep
    return out
