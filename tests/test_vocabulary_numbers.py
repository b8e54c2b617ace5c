"""Numbers that the kernels' fp32 cannot hold are refused (CPU)."""

from __future__ import annotations

import math

import pytest
import torch

from thundersync_amd import embedding


@pytest.mark.parametrize("scale", [1e39, -1e300, math.inf, math.nan])
def test_embedding_scale(scale):
    with pytest.raises(ValueError, match="scale must be a finite number"):
        embedding.embedding(torch.zeros(3, dtype=torch.int64), torch.zeros(8, 4), scale=scale)
