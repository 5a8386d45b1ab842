"""LowRankAdapters keeps copies: what its caller does to a, b and scaling afterwards is no matter."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def test_tensors_overwritten_after_construction(gpu_dev):
    import int_crush_converter_amd as icq
    g = torch.Generator().manual_seed(4)
    K, N, R = 200, 48, 8
    w = icq.QuantizedWeight(torch.randint(-128, 128, (N, K), generator=g).to(torch.int8).to(gpu_dev), torch.full((N,), 0.01, device=gpu_dev))
    for n in (3, 1):
        act = icq.quantize_activations(torch.randn(30, K, generator=g).to(gpu_dev))
        groups = icq.group_rows(torch.randint(0, n, (30,), generator=g).to(gpu_dev), n)
        a, b = torch.randn(n, R, K, generator=g).to(BF16).to(gpu_dev), torch.randn(n, N, R, generator=g).to(BF16).to(gpu_dev)
        scaling = torch.rand(n, generator=g).to(gpu_dev) + 0.5
        ad = icq.LowRankAdapters(a, b, scaling)
        y = icq.quantized_linear(act, w, adapters=ad, groups=groups)
        for t in (a, b, scaling):
            t.fill_(9.0)
        assert torch.equal(icq.quantized_linear(act, w, adapters=ad, groups=groups), y)
