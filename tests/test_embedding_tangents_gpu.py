"""Forward-mode derivatives of the embedding: a table's tangent reaches the rows, with and without gradients."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

from thundersync_amd.embedding import HipEmbedding, embedding

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("needs_grad", [False, True])
@pytest.mark.parametrize("scale", [1.0, 8.0])
def test_the_rows_carry_the_tables_tangent(cuda, dtype, needs_grad, scale):
    """The lookup is linear: the tangent is the tangent's lookup, the padding row's too (as torch has it)."""
    g = torch.Generator(device=cuda).manual_seed(0)
    table = torch.randn(30, 24, generator=g, device=cuda).to(dtype).requires_grad_(needs_grad)
    tangent = torch.randn(30, 24, generator=g, device=cuda).to(dtype)
    ids = torch.randint(0, 30, (5, 7), generator=g, device=cuda)
    with fwd.dual_level():
        out = fwd.unpack_dual(embedding(ids, fwd.make_dual(table, tangent), scale=scale, padding_idx=3))
        assert torch.equal(out.primal, embedding(ids, table, scale=scale)) and out.tangent is not None
        assert torch.equal(out.tangent, embedding(ids, tangent, scale=scale))
        with torch.no_grad():
            assert torch.equal(fwd.unpack_dual(embedding(ids, fwd.make_dual(table, tangent), scale=scale)).tangent,
                               out.tangent)
        assert fwd.unpack_dual(embedding(ids, table, scale=scale)).tangent is None


def test_of_the_module(cuda):
    """Against torch's own, the rows' tangents bit by bit."""
    plain = torch.nn.Embedding(20, 16, padding_idx=2, device=cuda)
    hip = HipEmbedding(20, 16, padding_idx=2, device=cuda)
    ids = torch.arange(20, device=cuda).flip(0)
    tangent = torch.randn(20, 16, device=cuda)
    got = []
    for module in (plain, hip):
        weight = plain.weight.detach()
        del module._parameters["weight"]
        with fwd.dual_level():
            module.weight = fwd.make_dual(weight, tangent)
            got.append(fwd.unpack_dual(module(ids)).tangent)
    assert torch.equal(*got)
