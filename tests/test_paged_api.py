"""Refusals of the paged cache, appending to it and attention over it, without a GPU."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from thundersync_amd import _lib
from thundersync_amd._abi import PagedBatch, PagedCacheDesc
from thundersync_amd.paged import CODES, PagedCache, append_tokens, paged_attention, rotary_table, stored_row

BF = torch.bfloat16


def pages(dtype=BF, shape=(4, 2, 16, 64)):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("key, value, scales, options, error, words", [
    (pages()[0], pages()[0], (), {}, ValueError, r"must be \[pages"),
    (pages(), pages(shape=(5, 2, 16, 64)), (), {}, ValueError, r"must be \[pages"),
    (pages(shape=(4, 2, 16, 80)),) * 2 + ((), {}, ValueError, "rows of 64, 128, 192, 256"),
    (pages(shape=(4, 2, 24, 64)),) * 2 + ((), {}, ValueError, "page_size must be one of"),
    (pages(shape=(4, 2, 512, 64)),) * 2 + ((), {}, ValueError, "page_size must be one of"),
    (pages(shape=(0, 2, 16, 64)),) * 2 + ((), {}, ValueError, "at least one page"),
    (pages(), pages(torch.float16), (), {}, TypeError, "must both be"),
    (pages(torch.float32),) * 2 + ((), {}, TypeError, "must both be"),
    (pages(),) * 2 + ((), {"dtype": torch.float16}, TypeError, "stands for"),
    (pages(CODES),) * 2 + ((torch.ones(4, 2, 1),) * 2, {"dtype": torch.float32}, TypeError, "stands for"),
    (pages(),) * 2 + ((), {"head_dim": 72}, ValueError, "head_dim 72 in rows of 64"),
    (pages(),) * 2 + ((), {"head_dim": 30}, ValueError, "multiple of 8"),
    (pages(CODES),) * 2 + ((), {}, ValueError, "goes with float8_e4m3fn pages"),
    (pages(),) * 2 + ((torch.ones(4, 2, 1),) * 2, {}, ValueError, "goes with float8_e4m3fn pages"),
    (pages(CODES),) * 2 + ((torch.ones(4, 2, 2),) * 2, {}, ValueError, "key_scale must be contiguous"),
    (pages(CODES),) * 2 + ((torch.ones(4, 2, 1).double(),) * 2, {}, TypeError, "key_scale must be fp32"),
    (pages(CODES),) * 2 + ((torch.ones(4, 2, 1), torch.ones(4, 1, 2).transpose(1, 2)[:, :1]), {}, ValueError,
                           "value_scale must be contiguous"),
    (pages().transpose(0, 1),) * 2 + ((), {}, ValueError, "each page must be dense"),
    (pages(shape=(4, 16, 16, 64)).transpose(1, 2),) * 2 + ((), {}, ValueError, "each page must be dense"),
    (pages().expand(4, 2, 16, 64)[:1].expand(3, 2, 16, 64),) * 2 + ((), {}, ValueError, "each page must be dense"),
    (torch.zeros(4 * 2048 + 1, dtype=BF)[1:].view(4, 2, 16, 64),) * 2 + ((), {}, ValueError, "multiples of 16 bytes"),
    (pages().requires_grad_(),) * 2 + ((), {}, ValueError, "holds no gradients"),
])
def test_cache_refusals(key, value, scales, options, error, words):
    with pytest.raises(error, match=words):
        PagedCache(key, value, *scales, **options)


@pytest.mark.parametrize("options, error", [({"bits": 4}, ValueError), ({"dtype": torch.float32}, TypeError),
                                            ({"head_dim": 12}, ValueError), ({"head_dim": 264}, ValueError),
                                            ({"page_size": 8}, ValueError), ({"pages": 0}, ValueError)])
def test_empty_refusals(options, error):
    with pytest.raises(error):
        PagedCache.empty(**{"pages": 4, "page_size": 16, "kv_heads": 2, "head_dim": 64, "device": "cpu"} | options)


def test_a_cache_on_the_cpu():
    """It can be laid out there; nothing runs on it."""
    cache = PagedCache.empty(4, 16, 2, 72, bits=8, device="cpu")
    assert cache.row == 128 and cache.key.shape == (4, 2, 16, 128) and cache.key_scale.shape == (4, 2, 1)
    assert cache.bits == 8 and cache.dtype == BF and cache.head_dim == 72
    assert PagedCache.empty(4, 16, 2, 72, device="cpu").values()[0].shape == (4, 2, 16, 72)
    with pytest.raises(RuntimeError, match="on the GPU only"):
        cache.values()
    assert [stored_row(d) for d in (8, 64, 72, 128, 136, 192, 200, 256)] == [64, 64, 128, 128, 192, 192, 256, 256]


def test_rotary_table():
    t = rotary_table(70000, 32, base=1e6, device="cpu")
    assert t.shape == (70000, 32) and t.dtype == torch.float32
    angle = 69999 * 1e6 ** (-2 * 5 / 32)
    assert abs(t[69999, 5].item() - math.cos(angle)) <= 2.0 ** -24 and abs(t[69999, 21].item() - math.sin(angle)) <= 2.0 ** -24
    with pytest.raises(ValueError, match="even"):
        rotary_table(4, 3, device="cpu")


X, Q, TABLE, LENGTHS = (torch.zeros(3, 2, 64, dtype=BF), torch.zeros(3, 4, 64, dtype=BF),
                        torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32))
OFF = torch.arange(4, dtype=torch.int32)
BATCH = [
    ({"page_table": TABLE[0]}, ValueError, r"page_table must be \[B, W\]"),
    ({"lengths": LENGTHS[:2]}, ValueError, r"lengths \[B\]"),
    ({"page_table": TABLE[:2], "lengths": LENGTHS[:2]}, ValueError, "one row: 3 rows for 2 sequences"),
    ({"offsets": OFF[:3]}, ValueError, r"offsets must be \[B \+ 1\]"),
    ({"page_table": TABLE.long()}, TypeError, "page_table must be int32"),
    ({"lengths": LENGTHS.long()}, TypeError, "lengths must be int32"),
    ({"offsets": OFF.long()}, TypeError, "offsets must be int32"),
    ({}, RuntimeError, "on the GPU only"),
    ({"offsets": OFF}, RuntimeError, "on the GPU only"),
]


@pytest.mark.parametrize("change, error, words", [
    ({"key": X[0]}, ValueError, r"key must be \[T, heads, 64\]"),
    ({"value": X[..., :32]}, ValueError, r"value must be \[T, heads, 64\]"),
    ({"key": X.half()}, TypeError, "key must be torch.bfloat16"),
    ({"key": X[:, :1], "value": X[:, :1]}, ValueError, r"must be \[T, 2, 64\]"),
    ({"value": X[:2]}, ValueError, "key and value must be"),
    ({"key": torch.zeros(3, 2, 64, dtype=BF, requires_grad=True)}, RuntimeError, "key requires grad"),
    ({"query": Q[:2]}, ValueError, "query has 2 rows and key 3"),
    ({"query": Q.half()}, TypeError, "query must be torch.bfloat16"),
    ({"rotary": torch.zeros(9)}, ValueError, r"rotary must be \[P, R\]"),
    ({"rotary": torch.zeros(9, 24)}, ValueError, "multiple of 16"),
    ({"rotary": torch.zeros(9, 80)}, ValueError, "multiple of 16 up to 64"),
    ({"rotary": torch.zeros(9, 32).double()}, TypeError, "rotary must be fp32"),
    ({"positions": torch.zeros(2, dtype=torch.int32)}, ValueError, r"positions must be \[T\]"),
    ({"positions": torch.zeros(3)}, TypeError, "positions must be int32"),
    *BATCH,
])
def test_append_refusals(change, error, words):
    args = {"cache": PagedCache.empty(4, 16, 2, 64, device="cpu"), "page_table": TABLE, "lengths": LENGTHS, "key": X,
            "value": X} | change
    with pytest.raises(error, match=words):
        append_tokens(**args)


@pytest.mark.parametrize("change, error, words", [
    ({"query": Q[0]}, ValueError, r"query must be \[T, heads, 64\]"),
    ({"query": Q[:, :3]}, ValueError, "not a multiple of KV heads 2"),
    ({"query": Q[:, :0]}, ValueError, "not a multiple of KV heads 2"),
    ({"query": Q.float()}, TypeError, "query must be torch.bfloat16"),
    ({"query": torch.zeros(3, 4, 64, dtype=BF, requires_grad=True)}, RuntimeError, "query requires grad"),
    ({"scale": math.inf}, ValueError, "scale must be a finite number"),
    ({"scale": None}, ValueError, "scale must be a finite number"),
    *BATCH,
])
def test_attention_refusals(change, error, words):
    args = {"query": Q, "cache": PagedCache.empty(4, 16, 2, 64, device="cpu"), "page_table": TABLE, "lengths": LENGTHS,
            "scale": 0.1} | change
    with pytest.raises(error, match=words):
        paged_attention(**args)


def desc(**change):
    p = 4096
    d = dict(key=p, value=p, key_scale=None, value_scale=None, key_page_stride=2048, value_page_stride=2048, pages=4,
             page_size=16, kv_heads=2, head_dim=64, row=64, bits=16, dtype=_lib.TS_BF16) | change
    return ctypes.byref(PagedCacheDesc(*d.values()))


def batch(**change):
    d = dict(table=4096, lengths=4096, offsets=None, ld_table=2, width=2, seqs=3) | change
    return ctypes.byref(PagedBatch(*d.values()))


@pytest.mark.parametrize("cache, seqs, words", [
    (dict(key=None), {}, "null cache"), (dict(dtype=0), {}, "cache dtype 0"), (dict(bits=4), {}, "a cache of 4 bits"),
    (dict(bits=8), {}, "scales of a cache of 8 bits"), (dict(key_scale=4096, value_scale=4096), {}, "scales of a cache of 16"),
    (dict(row=96), {}, "rows of 96"), (dict(head_dim=60), {}, "head dim 60"), (dict(head_dim=72), {}, "head dim 72"),
    (dict(page_size=48), {}, "pages of 48"), (dict(page_size=512), {}, "pages of 512"), (dict(kv_heads=0), {}, "0 KV heads"),
    (dict(key_page_stride=2040), {}, "strides 2040"), (dict(value_page_stride=2056), {}, "2056"), (dict(key=4104), {}, "16-byte"),
    (dict(pages=-1), {}, "-1 pages"),
    ({}, dict(seqs=-1), "bad batch"), ({}, dict(seqs=(1 << 20) + 1), "bad batch"), ({}, dict(width=-1), "bad batch"),
    ({}, dict(seqs=4), "3 rows for 4 sequences"), ({}, dict(lengths=None), "null pointer"), ({}, dict(table=None), "null pointer"),
])
def test_the_c_entries_refuse(cache, seqs, words):
    """Before any launch."""
    lib, p = _lib.require_library(), ctypes.c_void_p(4096)
    c, b = desc(**cache), batch(**seqs)
    assert lib.ts_paged_append(c, b, 3, p, 256, 64, 4, p, p, 128, 64, p, 128, 64, None, 0, 0, 0, None, None) == 1
    assert words in lib.ts_hip_last_error().decode()
    assert lib.ts_paged_attention(c, b, 3, p, 256, 64, 4, 0.1, p, p, 1 << 40, None) == 1
    assert words in lib.ts_hip_last_error().decode()
    if cache:
        assert lib.ts_paged_values(c, p, p, None) == 1
        assert words in lib.ts_hip_last_error().decode()
    assert lib.ts_paged_attention_workspace(c, b, 3, 4) == 0


def test_the_c_entries_refuse_rows():
    lib, p, odd = _lib.require_library(), ctypes.c_void_p(4096), ctypes.c_void_p(4104)
    good = [desc(), batch(), 3, p, 256, 64, 4, p, p, 128, 64, p, 128, 64, None, 0, 0, 0, None, None]
    for at, value, words in ((3, None, "null pointer"), (3, odd, "16-byte"), (4, 252, "16-byte"), (8, None, "null pointer"),
                             (11, odd, "16-byte"), (16, 24, "rotation of 24"), (16, 80, "rotation of 80"),
                             (16, 32, "rotation of 32"), (6, -1, "-1 query heads")):
        args = list(good)
        args[at] = value
        assert lib.ts_paged_append(*args) == 1 and words in lib.ts_hip_last_error().decode(), (at, value)
    good = [desc(), batch(), 3, p, 256, 64, 4, 0.1, p, p, 1 << 40, None]
    for at, value, words in ((3, None, "null pointer"), (3, odd, "16-byte"), (5, 60, "16-byte"), (6, 3, "3 heads over 2"),
                             (6, 0, "0 heads over 2"), (8, None, "null pointer"), (7, math.inf, "scale")):
        args = list(good)
        args[at] = value
        assert lib.ts_paged_attention(*args) == 1 and words in lib.ts_hip_last_error().decode(), (at, value)
    good[0] = desc(pages=0)
    assert lib.ts_paged_attention(*good) == 1 and "without pages" in lib.ts_hip_last_error().decode()
    many = batch(offsets=4096)
    assert lib.ts_paged_attention(desc(), many, (1 << 31) - 1, p, 1 << 18, 64, 4096, 0.1, p, p, 1 << 62, None) == 1
    assert "too large" in lib.ts_hip_last_error().decode()
    assert lib.ts_paged_append(desc(), many, (1 << 31) - 1, p, 1 << 18, 64, 4096, p, p, 128, 64, p, 128, 64, None, 0, 0, 0, None,
                               None) == 1
    assert "too large" in lib.ts_hip_last_error().decode()
    assert lib.ts_paged_values(desc(), p, p, None) == 1 and "16-bit cache" in lib.ts_hip_last_error().decode()
