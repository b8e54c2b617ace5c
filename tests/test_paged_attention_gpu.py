"""Attention over a paged cache against the oracle in 64 bits, within bounds that count its roundings."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import paged as ref
from tests.paged_cases import excess, int32, offsets_of, random_cache
from thundersync_amd import dispatch
from thundersync_amd.paged import PagedCache, paged_attention

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def check(cuda, lengths, counts=None, *, heads=8, kv_heads=2, dim=128, page=32, bits=8, dtype=BF, seed=0, scale=None,
          query=None, loud=1.0):
    g = torch.Generator().manual_seed(seed)
    cache, table, dense = random_cache(g, lengths, page=page, heads=kv_heads, dim=dim, dtype=dtype, bits=bits, device=cuda)
    counts_ = [1] * len(lengths) if counts is None else counts
    total, scale = sum(counts_), dim ** -0.5 if scale is None else scale
    q = (loud * torch.randn(total, heads, dim, generator=g)).to(dtype) if query is None else query
    out = paged_attention(q.to(cuda), cache, table, int32(lengths, cuda), scale,
                          offsets=None if counts is None else offsets_of(counts, cuda))
    assert out.dtype == dtype and out.shape == q.shape
    got, at = out.double().cpu(), 0
    for s, n in enumerate(counts_):
        if lengths[s]:
            want, bound = ref.attention(q[at:at + n], *dense[s], scale, dtype)
            over = excess(got[at:at + n], want, bound)
            assert over <= 0, (s, lengths[s], n, over, bound.max().item())
        else:
            assert not bool(got[at:at + n].any())
        at += n


LENGTHS = [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 130, 255, 257, 300, 0, 513]


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("page", [16, 128])
def test_one_token_each(cuda, dtype, bits, page):
    check(cuda, LENGTHS, dtype=dtype, bits=bits, page=page)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("dim", [8, 64, 72, 96, 128, 160, 192, 200, 256])
def test_head_dims(cuda, dim, bits):
    check(cuda, [70, 1, 33], dim=dim, bits=bits, page=16)
    check(cuda, [70, 9, 133], [5, 9, 40], dim=dim, bits=bits, page=64, dtype=FP)


@pytest.mark.parametrize("heads, kv_heads", [(1, 1), (4, 4), (5, 1), (6, 2), (12, 2), (16, 1), (17, 1), (40, 8), (34, 1),
                                             (71, 1)])
@pytest.mark.parametrize("counts", [None, [1, 3, 2]])
def test_groups(cuda, heads, kv_heads, counts):
    check(cuda, [90, 200, 2], counts, heads=heads, kv_heads=kv_heads, dim=64, page=64)


@pytest.mark.parametrize("dtype, bits, dim", [(BF, 8, 128), (FP, 8, 64), (BF, 16, 256), (FP, 16, 128), (BF, 8, 192)])
@pytest.mark.parametrize("counts", [
    [1, 2, 5, 8, 3, 1], [16, 17, 33, 1, 64, 0], [130, 1, 70, 200, 0, 31],
])
def test_several_tokens(cuda, dtype, bits, dim, counts):
    """Some sequences new with their tokens, some far in; a sequence may have none this time."""
    lengths = [c + extra for c, extra in zip(counts, (0, 100, 17, 333, 64, 1))]
    check(cuda, lengths, counts, dtype=dtype, bits=bits, dim=dim, page=16, seed=3)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("counts", [None, [4], [150]])
def test_long(cuda, bits, counts):
    check(cuda, [9001], counts, heads=8, kv_heads=1, dim=128, page=64, bits=bits)


@pytest.mark.parametrize("lengths, counts", [([5000, 3, 0, 1200, 40], None), ([3000, 3000, 50], [1, 65, 50]),
                                             ([20, 4000], [20, 2])])
def test_uneven_sequences(cuda, lengths, counts):
    check(cuda, lengths, counts, heads=8, kv_heads=2, dim=64, page=16)


@pytest.mark.parametrize("loud, scale", [(30.0, None), (1e3, 0.5), (1.0, 0.0), (2.0, -0.1)])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_peaked_and_even_rows(cuda, loud, scale, dtype):
    check(cuda, [300, 40, 2000], None, loud=loud, scale=scale, dtype=dtype)
    check(cuda, [300, 40], [70, 4], loud=loud, scale=scale, dtype=dtype)


def test_many_sequences(cuda):
    g = torch.Generator().manual_seed(5)
    lengths = torch.randint(0, 60, (300,), generator=g).tolist()
    check(cuda, lengths, heads=4, kv_heads=1, dim=64, page=16)
    counts = [min(n, k) for n, k in zip(lengths, torch.randint(0, 4, (300,), generator=g).tolist())]
    check(cuda, lengths, counts, heads=4, kv_heads=1, dim=64, page=16)


@pytest.mark.parametrize("counts", [None, [3, 1], [40, 100]])
@pytest.mark.parametrize("bits", [8, 16])
def test_strided_rows(cuda, counts, bits):
    """Queries as a projection's transposed view gives them, a page table wider than its rows, pages apart."""
    g = torch.Generator().manual_seed(1)
    lengths = [100, 212]
    cache, table, dense = random_cache(g, lengths, page=16, heads=2, dim=64, dtype=BF, bits=bits, device=cuda)
    total = 2 if counts is None else sum(counts)
    q = torch.randn(4, total, 64, generator=g).to(BF).to(cuda).transpose(0, 1)
    wide = torch.zeros(2, table.shape[1] + 5, dtype=torch.int32, device=cuda)
    wide[:, :table.shape[1]] = table
    both = torch.zeros(cache.pages, 2, *cache.key.shape[1:], device=cuda).to(cache.key.dtype)
    both[:, 0], both[:, 1] = cache.key, cache.value
    apart = PagedCache(both[:, 0], both[:, 1], cache.key_scale, cache.value_scale, dtype=BF)
    off = None if counts is None else offsets_of(counts, cuda)
    want = paged_attention(q.contiguous(), cache, table, int32(lengths, cuda), 0.1, offsets=off)
    got = paged_attention(q, apart, wide[:, :table.shape[1]], int32([100, 7, 212, 7], cuda)[::2], 0.1, offsets=off)
    assert torch.equal(got, want)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("counts", [[4, 9], [60, 33]])
def test_what_a_row_does_not_see(cuda, bits, bad, counts):
    """NaN and infinite values and keys of later tokens (infinities in 16 bits only: e4m3 has none) reach no earlier row."""
    g = torch.Generator().manual_seed(2)
    lengths = [80, 201]
    for which in (0, 1):
        cache, table, dense = random_cache(g, lengths, page=16, heads=2, dim=64, dtype=BF, bits=bits, device=cuda)
        pages = (cache.key, cache.value)[which]
        n = counts[0]
        pos = lengths[0] - n // 2  # one of the new tokens
        x = pages.float()
        x[int(table[0, pos // 16]), :, pos % 16] = bad
        pages.copy_(x.to(pages.dtype))
        q = torch.randn(sum(counts), 4, 64, generator=g).to(BF)
        out = paged_attention(q.to(cuda), cache, table, int32(lengths, cuda), 0.1, offsets=offsets_of(counts, cuda))
        dense[0][which][pos] = math.nan
        want, bound = ref.attention(q[:n], *dense[0], 0.1, BF)
        rows = slice(0, pos - (lengths[0] - n))
        got = out[:n].double().cpu()
        assert excess(got[rows], want[rows], bound[rows]) <= 0
        seen = got[pos - (lengths[0] - n):]
        assert not bool(seen.isfinite().all())
        want, bound = ref.attention(q[n:], *dense[1], 0.1, BF)
        assert excess(out[n:], want, bound) <= 0


@pytest.mark.parametrize("counts", [None, [1, 2, 1, 5], [60, 40, 1, 70]])
@pytest.mark.parametrize("bits", [8, 16])
def test_bad_pages_give_nan(cuda, counts, bits):
    """Rows that see a key on a page that is none, or past the page table, are NaN, and no others."""
    g = torch.Generator().manual_seed(4)
    lengths = [70, 90, 33, 75]
    cache, table, dense = random_cache(g, lengths, page=32, heads=2, dim=64, dtype=BF, bits=bits, device=cuda)
    table[1, 1] = cache.pages
    table[2, 0] = -1
    given = int32([70, 90, 33, 32 * table.shape[1] + 1], cuda)
    n = [1] * 4 if counts is None else counts
    n = [min(a, b) for a, b in zip(n, lengths)]
    q = torch.randn(sum(n), 4, 64, generator=g).to(BF)
    out = paged_attention(q.to(cuda), cache, table, given, 0.1, offsets=None if counts is None else offsets_of(n, cuda))
    got = out.double().cpu().split(n)
    want, bound = ref.attention(q[:n[0]], *dense[0], 0.1, BF)
    assert excess(got[0], want, bound) <= 0
    assert bool(got[1].isnan().all()) and bool(got[2].isnan().all())
    sees = 32 * table.shape[1] + 1 - n[3] + torch.arange(n[3])
    assert bool(got[3][sees >= 75].isnan().all())  # 75 tokens are there, NaN behind them
    assert bool(got[3][sees < 75].isfinite().all())


@pytest.mark.parametrize("counts", [None, [2, 3], [60, 40]])
@pytest.mark.parametrize("bits", [8, 16])
def test_tables_of_no_pages(cuda, counts, bits):
    """Every key is past the table."""
    cache = PagedCache.empty(2, 16, 1, 64, bits=bits, device=cuda)
    n = sum(counts) if counts else 2
    table = torch.empty(2, 0, dtype=torch.int32, device=cuda)
    q = torch.ones(n, 2, 64, device=cuda, dtype=BF)
    out = paged_attention(q, cache, table, int32(counts or [1, 1], cuda), 0.1,
                          offsets=offsets_of(counts, cuda) if counts else None)
    assert bool(out.isnan().all())
    out = paged_attention(q, cache, table, int32([0, 0], cuda), 0.1, offsets=offsets_of(counts, cuda) if counts else None)
    assert bool((out == 0).all())


def test_rows_of_no_sequence(cuda):
    """Rows behind the last sequence, rows of sequences without keys, more new tokens than keys: zeros."""
    g = torch.Generator().manual_seed(6)
    cache, table, dense = random_cache(g, [40, 0, 2], page=16, heads=1, dim=64, dtype=BF, bits=8, device=cuda)
    q = torch.randn(12, 2, 64, generator=g).to(BF)
    for offsets in ([0, 3, 5, 9], [0, 3, 5, 12], [0, 0, 0, 0]):
        out = paged_attention(q.to(cuda), cache, table, int32([40, 0, 2], cuda), 0.1, offsets=int32(offsets, cuda))
        got = out.double().cpu()
        want = torch.zeros(12, 2, 64, dtype=torch.float64)
        bound = torch.zeros_like(want)
        if offsets[1]:
            want[:3], bound[:3] = ref.attention(q[:3], *dense[0], 0.1, BF)
            last = offsets[3]
            want[last - 2:last], bound[last - 2:last] = ref.attention(q[last - 2:last], *dense[2], 0.1, BF)
        assert excess(got, want, bound) <= 0


@pytest.mark.parametrize("n", [2, 50])
@pytest.mark.parametrize("skipped", [1, 40])
def test_rows_before_the_first_sequence(cuda, n, skipped):
    g = torch.Generator().manual_seed(16)
    cache, table, dense = random_cache(g, [60, 70], page=16, heads=1, dim=64, dtype=BF, bits=8, device=cuda)
    q = torch.randn(skipped + n + 5, 2, 64, generator=g).to(BF)
    out = paged_attention(q.to(cuda), cache, table, int32([60, 70], cuda), 0.1,
                          offsets=int32([skipped, skipped + n, skipped + n + 1], cuda)).double().cpu()
    want, bound = torch.zeros_like(out), torch.zeros_like(out)
    for s, rows in enumerate((slice(skipped, skipped + n), slice(skipped + n, skipped + n + 1))):
        want[rows], bound[rows] = ref.attention(q[rows], *dense[s], 0.1, BF)
    assert excess(out, want, bound) <= 0


def test_shared_pages(cuda):
    """Sequences that begin with the same pages."""
    g = torch.Generator().manual_seed(7)
    cache, table, dense = random_cache(g, [100], page=16, heads=2, dim=64, dtype=BF, bits=8, device=cuda)
    q = torch.randn(3, 4, 64, generator=g).to(BF)
    out = paged_attention(q.to(cuda), cache, table.repeat(3, 1), int32([100, 64, 9], cuda), 0.1).double().cpu()
    for i, n in enumerate((100, 64, 9)):
        want, bound = ref.attention(q[i:i + 1], dense[0][0][:n], dense[0][1][:n], 0.1, BF)
        assert excess(out[i], want[0], bound[0]) <= 0


def test_same_bits_every_time_and_counted(cuda):
    g = torch.Generator().manual_seed(8)
    lengths = [2000, 5, 700]
    cache, table, _ = random_cache(g, lengths, page=64, heads=2, dim=128, dtype=BF, bits=8, device=cuda)
    q = torch.randn(3, 8, 128, generator=g).to(BF).to(cuda)
    before = dispatch.attention_path_counts().get("hip_paged", 0)
    outs = [paged_attention(q, cache, table, int32(lengths, cuda), 0.1) for _ in range(4)]
    assert all(torch.equal(x, outs[0]) for x in outs[1:])
    assert dispatch.attention_path_counts()["hip_paged"] == before + 4


def test_pages_past_two_to_the_31_bytes(cuda):
    """Offsets of pages pass 32 bits: 5 GB of keys, the last pages read."""
    page, heads, dim = 256, 8, 128
    pages = 20000  # 256 KB a page
    key, value = (torch.zeros(pages, heads, page, dim, dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn)
                  for _ in range(2))
    scale = torch.ones(pages, heads, page // 16, device=cuda)
    g = torch.Generator().manual_seed(9)
    ids = [pages - 1, pages - 2, 9000]
    kv = [torch.randn(len(ids), heads, page, dim, generator=g).to(torch.float8_e4m3fn) for _ in range(2)]
    for i, p in enumerate(ids):
        key[p], value[p] = kv[0][i].to(cuda), kv[1][i].to(cuda)
    cache = PagedCache(key, value, scale, scale, dtype=BF)
    q = torch.randn(1, 16, dim, generator=g).to(BF)
    out = paged_attention(q.to(cuda), cache, int32([ids], cuda), int32([700], cuda), 0.1)
    dense = [x.double().transpose(1, 2).reshape(-1, heads, dim)[:700] for x in kv]
    want, bound = ref.attention(q, *dense, 0.1, BF)
    assert excess(out, want, bound) <= 0


@pytest.mark.parametrize("bits", [8, 16])
def test_captured_with_other_batches(cuda, bits):
    """A captured call reads lengths, offsets and pages anew at each replay: few rows and chunks, cut tiles and whole ones."""
    g = torch.Generator().manual_seed(17)
    cache, table, dense = random_cache(g, [2500, 300, 40, 900], page=32, heads=2, dim=128, dtype=BF, bits=bits, device=cuda)
    q = torch.randn(120, 4, 128, generator=g).to(BF).to(cuda)
    batches = [([2500, 300, 40, 900], [100, 5, 10, 5]), ([2400, 300, 1, 0], [1, 1, 1, 0]), ([30, 299, 40, 77], [20, 60, 40, 0]),
               ([2500, 300, 40, 900], [2, 3, 2, 113])]
    pages, lengths, offsets = table.clone(), int32(batches[0][0], cuda), offsets_of(batches[0][1], cuda)
    call = lambda: paged_attention(q, cache, pages, lengths, 0.1, offsets=offsets)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for n, counts in batches + batches[::-1]:
        lengths.copy_(int32(n, cuda))
        offsets.copy_(offsets_of(counts, cuda))
        out.fill_(7.0)
        graph.replay()
        eager = call()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        want, bound = torch.zeros(out.shape, dtype=torch.float64), torch.zeros(out.shape, dtype=torch.float64)
        at = 0
        for s, (length, count) in enumerate(zip(n, counts)):
            rows = slice(at, at + count)
            want[rows], bound[rows] = ref.attention(q[rows].cpu(), *(x[:length] for x in dense[s]), 0.1, BF)
            at += count
        assert excess(out, want, bound) <= 0
