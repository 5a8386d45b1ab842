"""ic_expert_linear with an order that names no row of the activations, which only a caller of the C ABI can give."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("rows,N", [(20, 40), (300, 260), (3000, 700)])
@pytest.mark.parametrize("top", [1, 3])
def test_rows_outside_the_activations_are_the_last(gpu_dev, bits, rows, N, top):
    import int_crush_converter_amd as icq
    import int_crush_converter_amd._native as nat
    g = torch.Generator().manual_seed(rows + top)
    K, E, tokens = 130, 2, rows // top
    rows = tokens * top
    act = icq.quantize_activations(torch.randn(tokens, K, generator=g).to(gpu_dev))
    q = torch.randint(-8, 8, (E, N, K), generator=g).to(torch.int8)
    pack = lambda w: (w[:, 0::2] & 15).view(torch.uint8) | ((w[:, 1::2] & 15) << 4).view(torch.uint8)      # noqa: E731
    w = icq.ExpertWeight([icq.QuantizedWeight((pack(q[e]) if bits == 4 else q[e]).to(gpu_dev), torch.ones(N, device=gpu_dev)) for e in range(E)])
    offsets = torch.tensor([0, rows // 3, rows], dtype=torch.int32, device=gpu_dev)
    order = torch.randint(0, rows, (rows,), generator=g).int()
    bad = torch.rand(rows, generator=g) < 0.2
    order[bad] = torch.tensor([-1, rows, 2 ** 31 - 1, -2 ** 31, -5], dtype=torch.int32)[torch.randint(0, 5, (rows,), generator=g)][bad]
    source = torch.where(bad, tokens - 1, order.clamp(0, rows - 1) // top).to(gpu_dev)
    order, y = order.to(gpu_dev), torch.empty(rows, N, device=gpu_dev)
    m = act.meta.data_ptr()
    nat.check(nat.lib().ic_expert_linear(act.data, act.data.shape[1], m, m + 4 * tokens, tokens, offsets, order, top, E, rows, w.tiles, bits,
                                         w.scales, w.scale_kind, None, None, 0, N, K, y, nat.DT_F32, N, nat.stream()), "ic_expert_linear")
    x = act.data[:, :K].double() * act.scales.double()[:, None]
    for e, (lo, hi) in enumerate(((0, rows // 3), (rows // 3, rows))):
        want = x[source[lo:hi]] @ q[e].double().T.contiguous().to(gpu_dev)
        assert ((y[lo:hi].double() - want).abs() <= want.abs() * 2.0 ** -21 + 1e-12).all()
