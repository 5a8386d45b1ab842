"""More rows than one axis of a launch has threads for: 2^26 of one wave each,
2^24 of four waves (about 55 GB of the GPU's memory)."""

from __future__ import annotations

import ctypes
import os

import pytest
import torch


def test_limit_on_the_host():
    from int_crush_converter_amd import _native as nat
    if not os.path.exists(nat.LIB_PATH):
        from int_crush_converter_amd import build
        build.build()
    nat.load(require_gpu=False)
    one = ctypes.c_void_p(16)          # an address that no refused call touches
    assert nat._lib.ic_quantize_rows(one, 0, 1 << 31, 64, 64, None, 0, None, 0, 1e-6, 1, one, 128, one, one, None, 0, None) == -3
    assert nat._lib.ic_row_sums_i8(one, 1 << 31, 64, 64, one, None) == -3


def check(q, want, K):
    """Codes of rows whose one value (column K - 1) is ``want``: its sign times 127, and everything else 0."""
    assert torch.equal(q.data[:, K - 1], (want.sign() * 127).to(torch.int8))
    assert torch.equal(q.sums, want.sign().to(torch.int32) * 127)
    scales = (torch.arange(126).float().clamp(min=1e-30) / 127).to(want.device)       # (divided on the CPU: rounded correctly)
    assert torch.equal(q.scales, scales[want.abs().long()])
    assert int(torch.count_nonzero(q.data)) == int(torch.count_nonzero(want))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,K", [((1 << 26) + 5, 1), ((1 << 24) + 3, 1025)])
def test_quantise(gpu_dev, rows, K):
    import int_crush_converter_amd as icq
    torch.cuda.empty_cache()
    want = (torch.arange(rows, device=gpu_dev) % 251 - 125).to(torch.bfloat16)
    x = torch.zeros(rows, K, dtype=torch.bfloat16, device=gpu_dev)
    x[:, K - 1] = want
    q = icq.quantize_activations(x)
    check(q, want, K)
    del x, q
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_sums_of_codes(gpu_dev):
    import int_crush_converter_amd as icq
    torch.cuda.empty_cache()
    rows = (1 << 26) + 5
    codes = (torch.arange(rows, device=gpu_dev) % 255 - 127).to(torch.int8)[:, None]
    q = icq.QuantizedActivations.from_codes(codes, torch.ones(rows, device=gpu_dev))
    assert torch.equal(q.sums, codes[:, 0].int())
    del q
    torch.cuda.empty_cache()
