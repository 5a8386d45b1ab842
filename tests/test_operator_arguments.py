"""Arguments that are refused before the GPU is asked for anything."""

from __future__ import annotations

import pytest
import torch

import int_crush_converter_amd as icq


@pytest.mark.parametrize("width,K", [(0, None), (0, 0), (0, -1), (4, -3), (4, 0)])
def test_packed_rows_without_columns(width, K):
    codes = torch.zeros(2, width, dtype=torch.uint8)
    with pytest.raises(ValueError, match="in_features"):
        icq.Mxfp4Tensor.from_packed(codes, torch.zeros(2, 0, dtype=torch.uint8), in_features=K)
