"""The embedding's two passes by themselves refuse what their kernels cannot read (CPU)."""

from __future__ import annotations

import pytest
import torch

from thundersync_amd.embedding import HipEmbedding, embedding_backward, embedding_forward

IDS = torch.zeros(3, dtype=torch.int64)


@pytest.mark.parametrize("ids, rows", [
    (IDS, torch.zeros(3, 4)),
    (IDS, torch.zeros(3, 4, device="meta")),
    (IDS.to("meta"), torch.zeros(3, 4)),
])
def test_tensors_elsewhere(ids, rows):
    with pytest.raises(RuntimeError, match="runs on the GPU only"):
        embedding_forward(ids, rows, 1.0)
    with pytest.raises(RuntimeError, match="runs on the GPU only"):
        embedding_backward(ids, rows, 10)


def test_a_table_without_columns_is_torchs():
    assert HipEmbedding(5, 0)(IDS).shape == (3, 0)
