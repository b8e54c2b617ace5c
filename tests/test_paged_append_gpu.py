"""Appending to a paged cache against the oracle: places, rotation, blocks' scales and codes."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import paged as ref
from tests.paged_cases import excess, int32, offsets_of
from thundersync_amd.paged import PagedCache, append_tokens, rotary_table

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


class Mirror:
    """What the oracle says a cache holds: values [pages, heads, page, dim], exponents, and how far they may be off."""

    def __init__(self, cache):
        self.dtype, self.bits, self.page = cache.dtype, cache.bits, cache.page_size
        self.values = [x.double().cpu() for x in cache.values()]
        self.off = [torch.zeros_like(x) for x in self.values]
        if self.bits == 8:
            self.exponents = [x.log2().round().int().cpu() for x in (cache.key_scale, cache.value_scale)]

    def append(self, table, start, rows, slack):
        """rows (key, value) [n, heads, dim] in fp64 at positions start ..; slack: how far fp32 has the key rows off."""
        table = table.cpu()
        for x, (values, off) in enumerate(zip(self.values, self.off)):
            n, at = len(rows[x]), 0
            while at < n:
                pos = start + at
                page, slot = int(table[pos // self.page]), pos % self.page
                first = slot % 16
                count = min(16 - first, n - at)
                lines = slice(slot - first, slot - first + 16)
                for h in range(values.shape[1]):
                    new, extra = rows[x][at:at + count, h], slack[at:at + count, h] if x == 0 else 0.0
                    if self.bits == 16:
                        values[page, h, slot:slot + count] = new
                        off[page, h, slot:slot + count] = new.abs() * torch.finfo(self.dtype).eps / 2 + extra \
                            if x == 0 else 0.0
                        continue
                    b = (slot - first) // 16
                    got, e = ref.append_block(values[page, h, lines], int(self.exponents[x][page, h, b]), new, first,
                                              self.dtype)
                    old = self.exponents[x][page, h, b].item()
                    values[page, h, lines], self.exponents[x][page, h, b] = got, e
                    if e != old:  # values of slots without tokens go with the scale
                        values[page, h, slot + count:slot - first + 16] *= 2.0 ** (e - old)
                at += count

    def check(self, cache):
        if self.bits == 8:
            for e, scale in zip(self.exponents, (cache.key_scale, cache.value_scale)):
                assert torch.equal(scale.cpu().log2(), e.float())
        for values, off, got, name in zip(self.values, self.off, cache.values(), ("key", "value")):
            # a rotated key that fp32 rounds over a code's border goes to the next code: a step, for the few that lie there
            step = values.abs() * 2.0 ** -3 + 2.0 ** -9 if self.bits == 8 and name == "key" else off
            over = excess(got, values, step)
            assert over <= 0, (name, over)
            if self.bits == 8:
                d = (got.double().cpu() - values).abs()
                assert (d > 0).sum().item() <= (0 if name == "value" else 2 + d.numel() * 1e-4)


def turned(x, table, positions, interleaved):
    """Rows rotated in 64 bits and how far fp32's products and sums (three roundings of the terms) have them off."""
    if table is None:
        return x.double(), torch.zeros_like(x.double())
    size = ref.rotate(x.double().abs(), table.double().abs() * torch.tensor(1.0), positions, interleaved).abs()
    other = x.double().abs().amax(dim=-1, keepdim=True)
    return ref.rotate(x, table, positions, interleaved), 3 * 2.0 ** -24 * (size + 2 * other)


def run(cuda, steps, *, heads=4, kv_heads=2, dim=64, page=16, bits=8, dtype=BF, rotary=None, interleaved=False, seed=0,
        loud=1.0, shuffled=None):
    """Sequences that grow by steps (a list of counts each), checked after every call."""
    g = torch.Generator().manual_seed(seed)
    b = len(steps[0])
    most = [sum(s[i] for s in steps) for i in range(b)]
    width = max(-(-n // page) for n in most) + 1
    pages = b * width + 2
    cache = PagedCache.empty(pages, page, kv_heads, dim, dtype=dtype, bits=bits, device=cuda)
    table = torch.randperm(pages, generator=g)[:b * width].view(b, width).to(torch.int32).to(cuda)
    angles = None if rotary is None else rotary_table(max(most) + 5, rotary, base=1e4, device=cuda)
    mirror, lengths = Mirror(cache), [0] * b
    for k, counts in enumerate(steps):
        t = sum(counts)
        q, key, value = (torch.randn(t, h, dim, generator=g) * loud ** k for h in (heads, kv_heads, kv_heads))
        q, key, value = q.to(dtype), key.to(dtype), value.to(dtype)
        lengths = [n + c for n, c in zip(lengths, counts)]
        positions = torch.cat([torch.arange(n - c, n) for n, c in zip(lengths, counts)])
        given = None
        if shuffled is not None:
            positions = torch.randint(0, max(most) + 5, (t,), generator=g)
            given = positions.to(torch.int32).to(cuda)
        out = append_tokens(cache, table, int32(lengths, cuda), key.to(cuda), value.to(cuda), query=q.to(cuda),
                            offsets=None if counts == [1] * b else offsets_of(counts, cuda), rotary=angles,
                            positions=given, interleaved=interleaved)
        cpu = None if angles is None else angles.cpu()
        want, slack = turned(q, cpu, positions, interleaved)
        half = torch.finfo(dtype).eps / 2
        over = excess(out, want, want.abs() * half + slack + 2.0 ** -25)
        assert over <= 0, over
        want, slack = turned(key, cpu, positions, interleaved)
        at = 0
        for s, c in enumerate(counts):
            mirror.append(table[s], lengths[s] - c, (want[at:at + c], value[at:at + c].double()),
                          slack[at:at + c] + 2.0 ** -25)
            at += c
        mirror.check(cache)
    return cache


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("rotary", [None, 64])
def test_prompts_then_tokens(cuda, bits, dtype, rotary):
    run(cuda, [[5, 40, 16], [1, 1, 1], [1, 1, 1], [13, 3, 1], [1, 1, 1]], bits=bits, dtype=dtype, rotary=rotary)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("dim, rotary", [(64, 16), (64, 32), (80, 80), (128, 128), (128, 32), (192, 192), (256, 64),
                                         (256, 256), (8, None), (72, 16), (200, 48)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_head_dims(cuda, bits, dim, rotary, interleaved):
    run(cuda, [[17, 3], [1, 1]], bits=bits, dim=dim, rotary=rotary, interleaved=interleaved, page=32, dtype=FP)


@pytest.mark.parametrize("heads, kv_heads", [(1, 1), (32, 8), (24, 4), (7, 7)])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_heads_and_pages(cuda, heads, kv_heads, page):
    run(cuda, [[300, 1, 17], [1, 1, 1], [2, 40, 15]], heads=heads, kv_heads=kv_heads, page=page, rotary=32)


@pytest.mark.parametrize("loud", [30.0, 0.01])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_blocks_grow(cuda, loud, dtype):
    """Tokens of other sizes join a block: its scale grows with them and never shrinks."""
    run(cuda, [[3, 18], [1, 1], [1, 1], [2, 9]], loud=loud, dtype=dtype)


def test_rotation_by_given_positions(cuda):
    run(cuda, [[30, 5], [1, 1]], rotary=64, shuffled=True)
    run(cuda, [[30, 5], [1, 1]], rotary=64, shuffled=True, bits=16, interleaved=True)


def test_no_query_and_empty_calls(cuda):
    for bits in (8, 16):
        cache = PagedCache.empty(4, 16, 2, 64, bits=bits, device=cuda)
        x = torch.ones(3, 2, 64, dtype=BF, device=cuda)
        table = int32([[0, 1], [2, 3]], cuda)
        assert append_tokens(cache, table, int32([2, 1], cuda), x, 2 * x, offsets=int32([0, 2, 3], cuda)) is None
        key, value = cache.values()
        assert key.float().sum() == 3 * 128 and value.float().sum() == 2 * 3 * 128
        none = append_tokens(cache, table[:0], int32([], cuda), x[:0], x[:0], query=x[:0])
        assert none.shape == (0, 2, 64)
        append_tokens(cache, table, int32([2, 1], cuda), x[:0], x[:0], offsets=int32([0, 0, 0], cuda))
        assert torch.equal(cache.values()[0], key)


@pytest.mark.parametrize("bits", [8, 16])
def test_rows_that_go_nowhere(cuda, bits):
    """Padding, page ids that are none, positions past the table: the cache stays as it was and other sequences' tokens
    arrive; query rows of padding are zero."""
    cache = PagedCache.empty(6, 16, 1, 64, bits=bits, device=cuda)
    g = torch.Generator().manual_seed(0)
    x = torch.randn(5, 1, 64, generator=g).to(BF).to(cuda)
    table = int32([[0], [6], [-1], [3], [4]], cuda)
    q = append_tokens(cache, table, int32([1, 1, 1, 17, 0], cuda), x, x, query=x)
    key, _ = cache.values()
    key = key.float()
    assert key[0, 0, 0].abs().min() > 0 and key[0, 0, 1:].abs().max() == 0 and key[1:].abs().max() == 0
    assert torch.equal(q[:4], x[:4]) and q[4].abs().max() == 0
    # rows behind the last sequence, and more new tokens than the sequence has
    q = append_tokens(cache, int32([[1], [2]], cuda), int32([2, 1], cuda), x, x, query=x, offsets=int32([0, 2, 4], cuda))
    key = cache.values()[0].float()
    assert key[2, 0, 0].abs().min() > 0 and key[2, 0, 1:].abs().max() == 0 and key[3:].abs().max() == 0
    assert q[2].abs().max() == 0 and q[4].abs().max() == 0 and torch.equal(q[3], x[3])
    assert torch.equal(key[2, 0, 0], cache.values()[0].float()[2, 0, 0])


@pytest.mark.parametrize("bits", [8, 16])
def test_rows_before_the_first_sequence(cuda, bits):
    cache = PagedCache.empty(3, 16, 1, 64, bits=bits, device=cuda)
    x = torch.randn(9, 1, 64, generator=torch.Generator().manual_seed(1)).to(BF).to(cuda)
    q = append_tokens(cache, int32([[1], [2]], cuda), int32([10, 4], cuda), x, x, query=x, offsets=int32([3, 5, 8], cuda))
    assert q[:3].abs().max() == 0 and q[8].abs().max() == 0 and torch.equal(q[3:8], x[3:8])
    key = cache.values()[0].float()
    got = key.abs().amax(dim=(1, 3)) > 0  # [page, token]
    want = torch.zeros(3, 16, dtype=torch.bool)
    want[1, 8:10] = want[2, 1:4] = True
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("bits", [8, 16])
def test_numbers_that_are_none(cuda, bits):
    """NaN stays NaN; an infinity is NaN as a code, and neither moves the block's scale; positions past the table are NaN."""
    cache = PagedCache.empty(1, 16, 1, 64, bits=bits, device=cuda)
    x = torch.ones(2, 1, 64, dtype=BF, device=cuda)
    x[0, 0, 3], x[1, 0, 5] = math.nan, math.inf
    append_tokens(cache, int32([[0]], cuda), int32([2], cuda), x, x, offsets=int32([0, 2], cuda))
    key, _ = cache.values()
    assert bool(key[0, 0, 0, 3].isnan()) and not bool(key[0, 0, 1, 5].isfinite())
    ok = torch.ones(2, 64, dtype=torch.bool)
    ok[0, 3] = ok[1, 5] = False
    assert bool((key[0, 0, :2][ok.to(cuda)] == 1).all())
    y = torch.ones(1, 1, 64, dtype=BF, device=cuda)
    q = append_tokens(cache, int32([[0]], cuda), int32([9], cuda), y, y, query=y, rotary=rotary_table(8, 32, device=cuda))
    key, _ = cache.values()
    for row in (q[0, 0], key[0, 0, 8]):
        assert bool(row[:32].isnan().all()) and bool((row[32:] == 1).all())


@pytest.mark.parametrize("dtype, top", [(FP, 65504.0), (BF, 3.3895313892515355e38)])
def test_the_top_of_the_type(cuda, dtype, top):
    """Values that would round to the next power of two, which the type does not hold, stay finite."""
    cache = PagedCache.empty(1, 16, 1, 64, dtype=dtype, bits=8, device=cuda)
    x = torch.full((1, 1, 64), top, dtype=dtype, device=cuda)
    x[0, 0, ::2] = -x[0, 0, ::2]
    x[0, 0, 1] = top / 3
    append_tokens(cache, int32([[0]], cuda), int32([1], cuda), x, x)
    got = cache.values()[0][0, 0, 0].double().cpu()
    want = x[0, 0].double().cpu()
    assert excess(got, want, want.abs() * 2.0 ** -4) <= 0


def test_strided_rows(cuda):
    """Projections' transposed views, a slice of a fused projection, rows off a 16-byte border."""
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(9, 8, 64, generator=g).to(BF).to(cuda)
    odd = torch.randn(9 * 2 * 64 + 1, generator=g).to(BF).to(cuda)[1:].view(9, 2, 64)
    table, lengths, off = int32([[0, 1]], cuda), int32([20], cuda), int32([0, 9], cuda)
    angles = rotary_table(32, 64, device=cuda)
    for bits in (8, 16):
        got, want = (PagedCache.empty(2, 16, 2, 64, bits=bits, device=cuda) for _ in range(2))
        for key in (qkv[:, 4:6], odd, qkv[:, 4:6].transpose(0, 1).contiguous().transpose(0, 1)):
            a = append_tokens(got, table, lengths, key, qkv[:, 6:], query=qkv[:, :4], offsets=off, rotary=angles)
            b = append_tokens(want, table, lengths, key.contiguous(), qkv[:, 6:].contiguous(),
                              query=qkv[:, :4].contiguous(), offsets=off, rotary=angles)
            assert torch.equal(a, b)
            assert all(torch.equal(x, y) for x, y in zip(got.values(), want.values()))


def test_many_sequences(cuda):
    g = torch.Generator().manual_seed(4)
    counts = torch.randint(0, 5, (200,), generator=g).tolist()
    run(cuda, [counts, [1] * 200], heads=1, kv_heads=1, page=16, rotary=16)
