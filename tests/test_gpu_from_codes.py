"""Activations made of codes from elsewhere keep their own copy: what the
caller writes into its buffers afterwards changes no product, whatever the
width (the row sums that zero-points need are formed once)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("K", [128, 100, 1024, 1])
@pytest.mark.parametrize("rows", [1, 40])
def test_buffers_written_again(gpu_dev, rows, K):
    import int_crush_converter_amd as icq
    g = torch.Generator().manual_seed(K)
    codes = torch.randint(-128, 128, (rows, K), generator=g).to(torch.int8).to(gpu_dev)
    scales = torch.rand(rows, generator=g).to(gpu_dev)
    w = icq.QuantizedWeight(torch.randint(-128, 128, (48, K), generator=g).to(torch.int8).to(gpu_dev),
                            torch.full((48,), 0.01), torch.full((48,), 7, dtype=torch.int8))
    act = icq.QuantizedActivations.from_codes(codes, scales)
    y, c, s = icq.quantized_linear(act, w, out_dtype=torch.float32), codes.clone(), act.sums.clone()
    codes.fill_(3)
    scales.fill_(2)
    assert torch.equal(act.codes, c) and torch.equal(act.sums, s) and torch.equal(s.long(), c.long().sum(1))
    assert torch.equal(icq.quantized_linear(act, w, out_dtype=torch.float32), y)
    assert not act.data[:, K:].any()
