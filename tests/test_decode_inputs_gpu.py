"""A decoding step's operators over inputs at the edge of what they take: mixed id types, masks without rows, scales of blocks
that hold nothing, values at the lower end of fp16."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import logits as ref_logits
from oracle import paged as ref
from tests.paged_cases import excess, int32, offsets_of, random_cache
from tests.test_paged_attention_gpu import check
from thundersync_amd.logits import adjust_logits, pack_allowed
from thundersync_amd.paged import PagedCache, append_tokens, paged_attention, rotary_table

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


@pytest.mark.parametrize("history_ids, bias_ids", [(torch.int32, torch.int64), (torch.int64, torch.int32),
                                                   (torch.int64, torch.int64)])
def test_ids_past_32_bits_are_passed_over(cuda, history_ids, bias_ids):
    """Each list in its own type: an id of 64 bits that 32 would cut to a token is none."""
    vocab = 40
    far = [2 ** 32 + 5, -2 ** 63, -2 ** 32 + 6, 2 ** 31, 2 ** 63 - 1, 2 ** 32]
    near = [3, -1, vocab, vocab - 1, -2 ** 31, 2 ** 31 - 1]
    history = torch.tensor([near, near[::-1]] if history_ids == torch.int32 else [near, far]).to(history_ids)
    ids = torch.tensor([near, near] if bias_ids == torch.int32 else [far, near]).to(bias_ids)
    bias = torch.arange(1.0, 13.0).view(2, 6)
    z = torch.linspace(-2, 2, 2 * vocab).view(2, vocab)
    out = adjust_logits(z.to(cuda), history=history.to(cuda), presence=0.5, bias_ids=ids.to(cuda), bias=bias.to(cuda))
    want = torch.stack([ref_logits.adjust(z[i], history[i].tolist(), presence=0.5, bias_ids=ids[i].tolist(), bias=bias[i])
                        for i in range(2)])
    # a presence penalty and up to one bias of 12 on logits of up to 2: two roundings of less than 16
    assert excess(out, want, torch.full_like(want, 2 * 16 * 2.0 ** -24)) <= 0


@pytest.mark.parametrize("dtype", [BF, FP, torch.float32])
def test_rows_of_a_mask_without_rows(cuda, dtype):
    """No mask at all, and rows that name one: NaN, as past the last of several; rows that name none are as they were."""
    z = torch.randn(4, 70, generator=torch.Generator().manual_seed(0)).to(dtype).to(cuda)
    rows = int32([0, -1, 3, -5], cuda)
    empty = torch.empty(0, 3, dtype=torch.int32, device=cuda)
    out = adjust_logits(z, allowed=empty, allowed_rows=rows)
    assert bool(out[[0, 2]].isnan().all()) and torch.equal(out[[1, 3]], z[[1, 3]])
    out = adjust_logits(z, history=torch.zeros(4, 1, dtype=torch.int64, device=cuda), presence=1.0, allowed=empty,
                        allowed_rows=rows)
    assert bool(out[[0, 2]].isnan().all()) and torch.equal(out[[1, 3], 1:], z[[1, 3], 1:])


def with_stale_scales(cache, table, lengths):
    """The cache behind one more page, its first; that page's scales and those of blocks without tokens are NaN."""
    page, table = cache.page_size, table + 1
    first = lambda x, fill: torch.cat([torch.full_like(x[:1].float(), fill).to(x.dtype), x])  # noqa: E731
    held = torch.zeros(cache.pages + 1, 1, page // 16, dtype=torch.bool, device=table.device)
    for s, n in enumerate(lengths):
        for block in range(-(-n // 16)):
            held[int(table[s, block * 16 // page]), 0, block * 16 % page // 16] = True
    scales = [torch.where(held, first(x, math.nan), math.nan).contiguous() for x in (cache.key_scale, cache.value_scale)]
    codes = [first(x.view(torch.uint8), 0x7F).view(cache.key.dtype) for x in (cache.key, cache.value)]
    return PagedCache(*codes, *scales, dtype=cache.dtype, head_dim=cache.head_dim), table


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("counts", [None, [1] * 9, [1, 2, 3, 4, 1, 5, 2, 1, 3], [1, 15, 16, 3, 33, 40, 1, 60, 70]])
def test_scales_of_blocks_that_hold_nothing(cuda, dtype, page, counts):
    """Whatever the first page's scales and those behind a sequence's end hold, no row has part of it."""
    g = torch.Generator().manual_seed(11)
    lengths = [1, 15, 16, 17, 33, 48, 65, 144, 200]
    cache, table, dense = random_cache(g, lengths, page=page, heads=2, dim=64, dtype=dtype, bits=8, device=cuda)
    cache, table = with_stale_scales(cache, table, lengths)
    n = [1] * len(lengths) if counts is None else counts
    q = torch.randn(sum(n), 4, 64, generator=g).to(dtype)
    out = paged_attention(q.to(cuda), cache, table, int32(lengths, cuda), 0.1,
                          offsets=None if counts is None else offsets_of(counts, cuda))
    at = 0
    for s, c in enumerate(n):
        want, bound = ref.attention(q[at:at + c], *dense[s], 0.1, dtype)
        over = excess(out[at:at + c], want, bound)
        assert over <= 0, (s, lengths[s], c, over)
        at += c


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("loud", [2.0 ** -8, 2.0 ** -12, 2.0 ** -15, 2.0 ** -20])
def test_small_fp16_values_are_codes_of_fp16_values(cuda, loud, interleaved):
    """What a code stands for is a value of the type also where rotated keys lie below its smallest steps."""
    g = torch.Generator().manual_seed(12)
    cache = PagedCache.empty(4, 16, 2, 64, dtype=FP, bits=8, device=cuda)
    table, angles = int32([[2, 0, 3]], cuda), rotary_table(64, 64, device=cuda)
    key, value = (loud * torch.randn(40, 2, 64, generator=g) for _ in range(2))
    key, value = key.to(FP), value.to(FP)
    append_tokens(cache, table, int32([40], cuda), key.to(cuda), value.to(cuda), offsets=int32([0, 40], cuda),
                  rotary=angles, interleaved=interleaved)
    rows = ref.rotate(key, angles.cpu(), torch.arange(40), interleaved), value.double()
    for codes, scale, got, want in zip((cache.key, cache.value), (cache.key_scale, cache.value_scale), cache.values(), rows):
        scale = scale.double().cpu().repeat_interleave(16, dim=-1)[..., None]
        stands = codes.double().cpu() * scale
        assert torch.equal(stands, got.double().cpu())
        ids = table[0].long().cpu()
        flat = lambda x: x[ids].transpose(1, 2).flatten(0, 1)[:40]  # noqa: E731
        # half a step of a code, normal or below, and fp32's roundings of the rotation (three of up to twice the largest)
        bound = want.abs() * 2.0 ** -4 + flat(scale) * 2.0 ** -10 + 6 * 2.0 ** -24 * want.abs().amax(dim=-1, keepdim=True)
        assert excess(flat(got), want, bound) <= 0


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotated_keys_next_to_a_border_between_codes(cuda, dtype, interleaved):
    """Tables chosen so that half of the rotated elements lie within a rounding of a border: the code is that of the
    rotation rounded once to fp32, not of products that were rounded before."""
    g = torch.Generator().manual_seed(14)
    n, half = 400, 32
    sign = lambda *shape: 1.0 - 2.0 * torch.randint(0, 2, shape, generator=g)  # noqa: E731
    u, v = ((sign(n, half) * (0.5 + 0.5 * torch.rand(n, half, generator=g))).to(dtype) for _ in range(2))
    cos = 2 * torch.rand(n, half, generator=g) - 1
    # e4m3's borders below 1.5, for the scale 2^-6 that an element of 7 gives
    border = sign(n, half) * (8 + torch.randint(0, 8, (n, half), generator=g) + 0.5) * 2.0 ** -torch.randint(
        4, 6, (n, half), generator=g)
    sin = ((u.double() * cos.double() - border) / v.double()).float()
    key = torch.zeros(n, 1, 128, dtype=dtype)
    pair = (slice(0, 64, 2), slice(1, 64, 2)) if interleaved else (slice(0, half), slice(half, 64))
    key[:, 0, pair[0]], key[:, 0, pair[1]], key[:, 0, 100] = u, v, 7.0
    table = torch.cat([cos, sin], dim=1)
    cache = PagedCache.empty(25, 16, 1, 128, dtype=dtype, bits=8, device=cuda)
    append_tokens(cache, torch.arange(25, dtype=torch.int32, device=cuda)[None], int32([n], cuda), key.to(cuda), key.to(cuda),
                  offsets=int32([0, n], cuda), rotary=table.to(cuda), interleaved=interleaved)
    assert bool((cache.key_scale == 2.0 ** -6).all())
    want = ref.encode(ref.rotate(key, table, torch.arange(n), interleaved), -6, dtype)
    got = cache.values()[0].double().cpu().transpose(1, 2).flatten(0, 1)
    assert torch.equal(got, want), (got != want).sum()


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("counts, length", [(None, 30001), ([3], 30001), ([33], 30001), (None, 400), ([1], 400), ([3], 400),
                                            ([33], 400)])
def test_many_small_fp16_weights(cuda, counts, length, bits):
    """One key of score 17.5 before others of 0: each of these has a weight of 2^-25.2, together they are 30000 times that."""
    n = counts[0] if counts else 1
    row = torch.zeros(length, 1, 8, dtype=FP)
    key, value = row.clone(), row.clone() + 1.0
    key[3, 0, 0], value[3, 0, :4] = 7.0, 0.0
    cache = PagedCache.empty(length // 256 + 1, 256, 1, 8, dtype=FP, bits=bits, device=cuda)
    table = torch.arange(cache.pages, dtype=torch.int32, device=cuda)[None]
    lengths = int32([length], cuda)
    append_tokens(cache, table, lengths, key.to(cuda), value.to(cuda), offsets=int32([0, length], cuda))
    q = torch.zeros(n, 1, 8, dtype=FP)
    q[:, 0, 0] = 2.5
    out = paged_attention(q.to(cuda), cache, table, lengths, 1.0, offsets=None if counts is None else offsets_of(counts, cuda))
    others = (length - n + torch.arange(n, dtype=torch.float64)) * math.exp(-17.5)
    want = torch.ones(n, 1, 8, dtype=torch.float64)
    want[:, 0, :4] = (others / (1 + others))[:, None]
    # the result's half a step, the weights' (each within 2^-32 of the largest), fp32 sums of 30000
    bound = want * 2.0 ** -11 + length * 2.0 ** -32 + want * (length + 100) * 2.0 ** -24 + 2.0 ** -25
    assert excess(out, want, bound) <= 0


@pytest.mark.parametrize("kv_heads", [1, 4])
@pytest.mark.parametrize("kind", ["one", "few", "mixed"])
@pytest.mark.parametrize("bits", [8, 16])
def test_more_than_64_long_sequences(cuda, kv_heads, kind, bits):
    """The search for a work-group's borders goes over several 64s of sequences whose tiles are cut."""
    g = torch.Generator().manual_seed(13)
    lengths = torch.randint(600, 3001, (131,), generator=g).tolist()
    counts = None if kind == "one" else torch.randint(0, 4, (131,), generator=g).tolist()
    if kind == "mixed":
        for s in (0, 63, 64, 100, 130):
            counts[s] = 40
    check(cuda, lengths, counts, heads=2 * kv_heads, kv_heads=kv_heads, dim=64, page=64, bits=bits, seed=13)


def test_packing_a_mask_takes_little_memory(cuda):
    """The bits of a mask, of any width, in a few bytes a token."""
    g = torch.Generator(device=cuda).manual_seed(0)
    for rows, vocab in ((1, 1), (3, 31), (2, 64), (5, 1001), (200, 151936)):
        mask = torch.rand(rows, vocab, generator=g, device=cuda) < 0.5
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        bits = pack_allowed(mask)
        used = torch.cuda.max_memory_allocated() - before
        assert bits.dtype == torch.int32 and bits.shape == (rows, -(-vocab // 32))
        back = (bits[..., None] >> torch.arange(32, device=cuda, dtype=torch.int32)) & 1
        assert torch.equal(back.flatten(1)[:, :vocab].bool(), mask) and not bool(back.flatten(1)[:, vocab:].any())
        assert used <= 3 * mask.numel() + 65536, used / mask.numel()


def test_checked_batches_with_rows_of_no_sequence(cuda, monkeypatch):
    """The check of a batch lets pass what the module describes: rows outside the sequences, padding with rows of its own."""
    monkeypatch.setenv("THUNDERSYNC_CHECK_TARGETS", "1")
    x = torch.ones(9, 1, 64, dtype=BF, device=cuda)
    table, lengths, offsets = int32([[0, 1], [2, 3], [9, 9]], cuda), int32([17, 3, 0], cuda), int32([2, 4, 5, 7], cuda)
    cache = PagedCache.empty(4, 16, 1, 64, device=cuda)
    q = append_tokens(cache, table, lengths, x, x, query=x, offsets=offsets)
    out = paged_attention(x, cache, table, lengths, 1.0, offsets=offsets)
    for rows in (q, out):
        assert not bool(rows[[0, 1, 5, 6, 7, 8]].any()) and bool((rows[2:5] != 0).all())
    for bad in ([-1, 4, 5, 7], [2, 4, 3, 7], [2, 4, 5, 10]):
        with pytest.raises(ValueError, match="offsets"):
            paged_attention(x, cache, table, lengths, 1.0, offsets=int32(bad, cuda))
