"""The paged cache's and the logits' oracles against torch's own operations and hand-worked values (CPU)."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import logits as ref_logits
from oracle import paged as ref


@pytest.mark.parametrize("most, exponent", [(448.0, 0), (448.5, 1), (447.0, 0), (224.0, -1), (224.25, 0), (1.75, -8),
                                            (1.0, -8), (0.0, -118), (1e-40, -118), (65504.0, 8), (3.3e38, 120)])
def test_exponents(most, exponent):
    assert ref.exponent_for(most) == exponent
    if 1e-30 < most < 1e38:
        assert most <= 448.0 * 2.0 ** exponent and most > 448.0 * 2.0 ** (exponent - 1)


def test_codes_are_values_of_both_types():
    g = torch.Generator().manual_seed(0)
    for dtype, scale in ((torch.bfloat16, 1e30), (torch.float16, 65504.0), (torch.float16, 1e-6), (torch.bfloat16, 3.38e38)):
        x = (torch.randn(64, generator=g).clamp(-1, 1) * scale).to(dtype)
        x[0] = torch.finfo(dtype).max if scale > 1e38 or scale == 65504.0 else x[0]
        e = ref.exponent_for(float(x.double().abs().max()))
        y = ref.encode(x, e, dtype)
        assert torch.equal(y.to(dtype).double(), y) and bool(y.to(dtype).isfinite().all())
        assert bool(((y - x.double()).abs() <= x.double().abs() * 2.0 ** -4 + 2.0 ** (e - 10)).all())


def test_a_growing_block_keeps_its_values():
    g = torch.Generator().manual_seed(1)
    new = torch.randn(16, 64, generator=g).to(torch.bfloat16)
    block, e = ref.append_block(torch.zeros(16, 64, dtype=torch.float64), ref.MIN_EXPONENT, new[:5], 0, torch.bfloat16)
    grown, e2 = ref.append_block(block, e, new[5:9] * 64, 5, torch.bfloat16)
    assert e2 >= e + 4
    far = block[:5].abs() >= 2.0 ** (e2 - 6)  # normal codes by the new scale
    assert far.any() and torch.equal(grown[:5][far], block[:5][far]) and torch.equal(grown[9:], block[9:])


def test_rotation():
    x = torch.zeros(2, 1, 4)
    x[:, 0, 0] = 1.0
    table = torch.tensor([[1.0, 1.0, 0.0, 0.0], [0.0, 1.0, 1.0, 0.0]])
    assert ref.rotate(x, table, torch.tensor([0, 1]))[:, 0].tolist() == [[1, 0, 0, 0], [0, 0, 1, 0]]
    assert ref.rotate(x, table, torch.tensor([0, 1]), True)[:, 0].tolist() == [[1, 0, 0, 0], [0, 1, 0, 0]]


@pytest.mark.parametrize("n, length, heads, hkv", [(1, 1, 2, 1), (1, 9, 4, 2), (3, 7, 2, 2), (5, 5, 6, 2)])
def test_attention(n, length, heads, hkv):
    g = torch.Generator().manual_seed(2)
    q = torch.randn(n, heads, 8, generator=g, dtype=torch.float64)
    k, v = (torch.randn(length, hkv, 8, generator=g, dtype=torch.float64) for _ in range(2))
    out, bound = ref.attention(q, k, v, 0.3, torch.bfloat16)
    k, v = (x.repeat_interleave(heads // hkv, dim=1).transpose(0, 1) for x in (k, v))
    mask = torch.arange(length) <= (length - n + torch.arange(n))[:, None]
    want = torch.nn.functional.scaled_dot_product_attention(q.transpose(0, 1), k, v, attn_mask=mask, scale=0.3)
    assert torch.allclose(out, want.transpose(0, 1), rtol=1e-12) and bool((bound >= 0).all())


def test_rows_without_keys_are_zero():
    out, _ = ref.attention(torch.ones(2, 1, 8), torch.ones(1, 1, 8), torch.ones(1, 1, 8), 1.0, torch.bfloat16)
    assert out[0].abs().max() == 0 and out[1].min() == 1


def test_logits():
    z = ref_logits.adjust([2.0, -2.0, 1.0, 0.5, 3.0], history=[0, 1, 4, 4, -1, 9], prompt=2, repetition=2.0, frequency=0.5,
                          presence=1.0, bias_ids=[2, 2, -1], bias=[1.0, 0.25, 7.0], allowed=[1, 1, 1, 0, 1])
    assert z.tolist() == [1.0, -4.0, 2.25, -math.inf, 1.5 - 1.0 - 1.0]
