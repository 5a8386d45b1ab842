"""Operands that lie on another GPU than the current one, or in host memory, are
refused before anything is launched.  No GPU: the tensors are stand-ins and
the library's calls are recorded instead of made."""

from __future__ import annotations

import pytest
import torch

from int_crush_converter_amd import _native as nat
from int_crush_converter_amd import activations, linear, mxfp4


class On:
    """What a tensor in the memory of GPU ``index`` (-1: the host) answers."""

    def __init__(self, index, *shape, dtype=torch.uint8):
        self.index, self.shape, self.dtype, self.is_cuda = index, torch.Size(shape), dtype, index >= 0
        self.device = torch.device("cuda", index) if index >= 0 else torch.device("cpu")

    def get_device(self):
        return self.index

    def data_ptr(self):
        return 4096


@pytest.fixture
def calls(monkeypatch):
    made = []
    for mod in (activations, linear, mxfp4):
        monkeypatch.setattr(mod, "call", lambda name, *args: made.append(name))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(nat, "_raw_stream", lambda dev: 0)
    monkeypatch.setattr(nat, "dtype_code", lambda t: 1)
    monkeypatch.setattr(torch, "empty", lambda size, dtype, device: On(device.index if device.index is not None else -1, *size))
    return made


def integer(i, meta=None):
    return activations.QuantizedActivations._of(On(i, 3, 128), On(i if meta is None else meta, 2, 3), 100, (3,))


def weight(i, scales=None, zeros=None):
    w = linear.QuantizedWeight.__new__(linear.QuantizedWeight)
    w.tiles, w.scales, w.scale_kind, w.bits, w.in_features, w.out_features = On(i, 4096), On(i if scales is None else scales, 16), 0, 4, 100, 16
    w.zero_points = None if zeros is None else On(zeros, 16)
    return w


def mx(i, scales=None, rows=3):
    t = mxfp4.Mxfp4Tensor.__new__(mxfp4.Mxfp4Tensor)
    t.tiles, t.scales, t.in_features, t.lead, t.rows = On(i, 1024), On(i if scales is None else scales, 256), 100, (rows,), rows
    return t


@pytest.mark.parametrize("where", [1, -1])
def test_operands_elsewhere_are_refused(calls, where):
    refused = [
        lambda: linear.quantized_linear(integer(where), weight(where)),
        lambda: linear.quantized_linear(integer(where), weight(0)),
        lambda: linear.quantized_linear(integer(0), weight(where)),
        lambda: linear.quantized_linear(integer(0, meta=where), weight(0)),
        lambda: linear.quantized_linear(integer(0), weight(0, scales=where)),
        lambda: linear.quantized_linear(integer(0), weight(0, zeros=where)),
        lambda: mxfp4.mxfp4_linear(mx(where), mx(where)),
        lambda: mxfp4.mxfp4_linear(mx(where), mx(0)),
        lambda: mxfp4.mxfp4_linear(mx(0), mx(where)),
        lambda: mxfp4.mxfp4_linear(mx(0, scales=where), mx(0)),
        lambda: mxfp4.mxfp4_linear(mx(0), mx(0, scales=where)),
        lambda: integer(where).dequantize(),
        lambda: integer(0, meta=where).dequantize(),
        lambda: mx(where).dequantize(),
        lambda: mx(0, scales=where).dequantize(),
        lambda: mx(where).to_packed(),
        lambda: mx(0, scales=where).to_packed(),
    ]
    for f in refused:
        with pytest.raises(ValueError, match="current device is cuda:0"):
            f()
        assert not calls


def test_operands_on_the_current_gpu_are_taken(calls):
    linear.quantized_linear(integer(0), weight(0, zeros=0))
    mxfp4.mxfp4_linear(mx(0), mx(0))
    integer(0).dequantize()
    mx(0).dequantize()
    assert calls == ["ic_quantized_linear", "ic_mxfp4_linear", "ic_dequantize_rows", "ic_mxfp4_dequantize"]
