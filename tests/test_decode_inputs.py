"""Inputs of a decoding step's operators that need no GPU: what is refused, what a check of the batch lets pass."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch
from torch.autograd import forward_ad

from tests.paged_cases import int32
from thundersync_amd import _lib
from thundersync_amd._abi import PagedBatch, PagedCacheDesc
from thundersync_amd.logits import adjust_logits, pack_allowed
from thundersync_amd.paged import PagedCache, append_tokens, paged_attention

BF = torch.bfloat16


def test_an_output_of_one_column_has_rows_of_its_own():
    """One column, whose rows are one element: a kernel would write past it."""
    z = torch.zeros(3, 1)
    for out in (torch.empty(1, 1).expand(3, 1), torch.empty(1).expand(3)[:, None]):
        with pytest.raises(ValueError, match="out must have rows of their own"):
            adjust_logits(z, out=out)
    for out in (torch.empty(3, 1), torch.empty(3, 8)[:, 2:3], torch.empty(1, 3).t()):
        with pytest.raises(RuntimeError, match="on the GPU only"):
            adjust_logits(z, out=out)


def test_the_c_entry_refuses_masks_that_are_not_there():
    lib, p = _lib.require_library(), ctypes.c_void_p(4096)
    args = [p, 70, 3, 70, None, 0, 0, None, None, None, 1.0, None, 0.0, None, 0.0, None, 0, None, 0, 0, None, 0, p, 2, 8, p, 70,
            0, None]
    assert lib.ts_adjust_logits(*args) == 1 and "null pointer" in lib.ts_hip_last_error().decode()


def append(**change):
    x = torch.zeros(3, 2, 64, dtype=BF)
    return append_tokens(**{"cache": PagedCache.empty(4, 16, 2, 64, device="cpu"), "lengths": int32([1] * 3, "cpu"),
                            "page_table": torch.zeros(3, 2, dtype=torch.int32), "key": x, "value": x} | change)


def attend(**change):
    return paged_attention(**{"query": torch.zeros(3, 4, 64, dtype=BF), "cache": PagedCache.empty(4, 16, 2, 64, device="cpu"),
                              "page_table": torch.zeros(3, 2, dtype=torch.int32), "lengths": int32([1] * 3, "cpu"),
                              "scale": 0.1} | change)


def adjust(**change):
    return adjust_logits(**{"logits": torch.zeros(3, 70), "history": torch.zeros(3, 5, dtype=torch.int64)} | change)


ROWS = [(append, "key", (3, 2, 64), BF), (append, "value", (3, 2, 64), BF), (append, "query", (3, 4, 64), BF),
        (attend, "query", (3, 4, 64), BF), (adjust, "logits", (3, 70), torch.float32)]


@pytest.mark.parametrize("call, name, shape, dtype", ROWS)
def test_tangents_are_refused(call, name, shape, dtype):
    """A tangent would be lost without a word; torch.no_grad() does not switch it off, as in torch."""
    x = torch.zeros(shape, dtype=dtype)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match=f"{name} ha(s|ve) a forward-mode tangent"):
            call(**{name: dual})
        with torch.no_grad(), pytest.raises(RuntimeError, match=f"{name} ha(s|ve) a forward-mode tangent"):
            call(**{name: dual})
        with pytest.raises(RuntimeError, match="on the GPU only"):
            call(**{name: dual.detach()})
    with pytest.raises(RuntimeError, match="on the GPU only"):
        call(**{name: x})


@pytest.mark.parametrize("call, name, shape", [(append, "rotary", (9, 32)), (adjust, "bias", (3, 2)), (adjust, "repetition", (3,)),
                                               (adjust, "frequency", (3,)), (adjust, "presence", (3,)), (adjust, "out", (3, 70))])
def test_gradients_of_other_inputs_are_refused(call, name, shape):
    """Of a table, biases, penalties, an output: what would be dropped is refused as it is for rows and logits."""
    x = torch.ones(shape)
    more = {"bias_ids": torch.zeros(3, 2, dtype=torch.int64)} if name == "bias" else {}
    leaf = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match=f"{name} requires grad"):
        call(**{name: leaf}, **more)
    with torch.no_grad(), pytest.raises(RuntimeError, match="on the GPU only"):
        call(**{name: leaf}, **more)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match=f"{name} has a forward-mode tangent"):
        call(**{name: forward_ad.make_dual(x, x)}, **more)
    with pytest.raises(RuntimeError, match="on the GPU only"):
        call(**{name: x}, **more)


@pytest.mark.parametrize("bits", [8, 16])
def test_what_a_cache_was_made_of_is_not_set_anew(bits):
    """The kernels would go on with the tensors, sizes and types that they were given."""
    cache, other = (PagedCache.empty(4, 16, 2, 64, bits=bits, device="cpu") for _ in range(2))
    was = {name: getattr(cache, name) for name in sorted(PagedCache._GIVEN)}
    for name in was:
        with pytest.raises(AttributeError, match=f"{name} of a PagedCache"):
            setattr(cache, name, getattr(other, name))
        assert getattr(cache, name) is was[name]
    cache.owner = "a rollout"  # a program's own
    assert cache.owner == "a rollout" and cache._desc.key == cache.key.data_ptr()


@pytest.mark.parametrize("rows, vocab", [(1, 70), (3, 1), (1, 1)])
def test_an_output_that_is_the_logits_by_other_strides(rows, vocab):
    """A single row or column is the same whatever stride the tensor gives it."""
    x = torch.zeros(500)
    z = x.as_strided((rows, vocab), (80 if rows == 1 else 5, 1))
    out = x.as_strided((rows, vocab), (200 if rows == 1 else 5, 1 if vocab > 1 else 3))
    assert z.stride() != out.stride()
    with pytest.raises(RuntimeError, match="on the GPU only"):
        adjust_logits(z, out=out)


@pytest.mark.parametrize("rows, vocab", [(0, 40), (1, 1), (3, 31), (2, 32), (2, 33), (5, 1001), (64, 64)])
def test_packed_masks(rows, vocab):
    """Masks of any width, of no rows, seen as columns."""
    mask = torch.rand(rows, vocab, generator=torch.Generator().manual_seed(rows)) < 0.5
    for given in (mask, mask.t().contiguous().t()):
        bits = pack_allowed(given)
        assert bits.dtype == torch.int32 and bits.shape == (rows, -(-vocab // 32)) and bits.is_contiguous()
        back = ((bits[..., None] >> torch.arange(32, dtype=torch.int32)) & 1).flatten(1).bool()
        assert torch.equal(back[:, :vocab], mask) and not bool(back[:, vocab:].any())


@pytest.mark.parametrize("scale", [3e38, -2.5e38, math.inf, math.nan])
def test_scales_that_pass_fp32_in_log2_units_are_refused(scale):
    """They are infinite where the kernels use them, and every row would be NaN."""
    lib, p = _lib.require_library(), ctypes.c_void_p(4096)
    cache = ctypes.byref(PagedCacheDesc(4096, 4096, None, None, 2048, 2048, 4, 16, 2, 64, 64, 16, _lib.TS_BF16))
    batch = ctypes.byref(PagedBatch(4096, 4096, None, 2, 2, 3))
    # a workspace too small for any batch: the call ends at the host's checks whatever the scale
    assert lib.ts_paged_attention(cache, batch, 3, p, 256, 64, 4, scale, p, p, 0, None) == 1
    assert "scale" in lib.ts_hip_last_error().decode()
    assert lib.ts_paged_attention(cache, batch, 3, p, 256, 64, 4, 2e38, p, p, 0, None) == 1
    assert "workspace of 0 bytes" in lib.ts_hip_last_error().decode()
