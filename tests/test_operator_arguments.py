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


def test_activations_of_wrong_tensors():
    """The kernels read what the shapes promise, so a handle made by hand has to hold it."""
    i8 = lambda *s: torch.zeros(s, dtype=torch.int8)                                             # noqa: E731
    meta = torch.zeros(2, 3)
    icq.QuantizedActivations(i8(3, 128), meta, 100, (3,))
    icq.QuantizedActivations(i8(6, 256), torch.zeros(2, 6), 129, (2, 3))
    icq.QuantizedActivations(i8(0, 128), torch.zeros(2, 0), 100, (2, 0))
    for data, m, K, lead in ((i8(3, 100), meta, 100, (3,)), (i8(2, 128), meta, 100, (3,)), (i8(3, 128).float(), meta, 100, (3,)),
                             (i8(3, 128), torch.zeros(2, 8)[:, 2:5], 100, (3,)), (i8(3, 128), meta.double(), 100, (3,)),
                             (i8(3, 256)[:, :128], meta, 100, (3,)), (i8(3, 128), meta, 200, (3,)), (i8(3, 128), meta, 0, (3,)),
                             (i8(4 * 128)[8:8 + 3 * 128].reshape(3, 128), meta, 100, (3,)), (i8(3, 128), meta, 100, (1, 4))):
        with pytest.raises(ValueError):
            icq.QuantizedActivations(data, m, K, lead)


def test_mxfp4_of_wrong_tensors():
    u8 = lambda n: torch.zeros(n, dtype=torch.uint8)                                             # noqa: E731
    icq.Mxfp4Tensor(u8(2 * 2 * 1024), u8(2 * 256), 129, (17,), 17)
    icq.Mxfp4Tensor(u8(0), u8(0), 129, (0, 5), 0)
    for tiles, scales, K, lead, rows in ((u8(3 * 1024), u8(512), 129, (17,), 17), (u8(4096), u8(256), 129, (17,), 17),
                                         (u8(4096), u8(512), 129, (16,), 17), (u8(4096), u8(512), 0, (17,), 17),
                                         (u8(4096).to(torch.int8), u8(512), 129, (17,), 17), (u8(8192)[::2], u8(512), 129, (17,), 17),
                                         (u8(5000)[8:4104], u8(512), 129, (17,), 17)):
        with pytest.raises(ValueError):
            icq.Mxfp4Tensor(tiles, scales, K, lead, rows)
