"""Inputs of a decoding step's operators that need no GPU: what is refused, what a check of the batch lets pass."""

from __future__ import annotations

import ctypes

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from tests.paged_cases import int32
from thundersync_amd import _lib, paged
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
