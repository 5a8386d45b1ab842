"""The norm of rows whose squares leave fp32's range, upwards or downwards,
against 64 bits, with the bounds of test_gpu_activations (the norm's value is
of ordinary size whatever the row's)."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_activations import BF16, F16, F32, check, exact

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("K,rot", [(64, 0), (1000, 64), (1024, 256), (4096, 256), (12288, 0), (20480, 64), (65536, 0)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_large_rows(gpu_dev, K, rot, dtype):
    """Rows of 1e18 (whose sum still fits where it is short), 1e20, 1e30 and near the largest value, ordinary rows between."""
    import int_crush_converter_amd as icq
    g = torch.Generator().manual_seed(K)
    size = torch.tensor([1.0, 1e18, 1e20, 1e-3, 1e30, 5e37, 1e19])[:, None]
    x = (torch.randn(7, K, generator=g).clamp(-4, 4) * size).to(dtype)
    r = (torch.randn(7, K, generator=g).clamp(-4, 4) * size * 0.1).to(dtype)
    w = (1 + 0.2 * torch.randn(K, generator=g)).to(dtype)
    for residual in (None, r):
        h, z = exact(x, w, residual, 1e-6, rot)
        q, out = icq.rms_norm_quantize(x.to(gpu_dev), w.to(gpu_dev), None if residual is None else residual.to(gpu_dev),
                                       rot_size=rot)
        check(q, z)
        if residual is not None:
            assert torch.equal(out.cpu(), (x.float() + r.float()).to(dtype))


@pytest.mark.parametrize("K,rot", [(64, 16), (1000, 0), (4096, 256), (20480, 0)])
@pytest.mark.parametrize("eps", [0.0, 1e-40, 1e-34, 1e-6])
def test_small_rows(gpu_dev, K, rot, eps):
    """Rows whose squares vanish: normalised where eps is 0 or as small, next to nothing where eps outweighs them."""
    import int_crush_converter_amd as icq
    g = torch.Generator().manual_seed(K)
    size = torch.tensor([1.0, 1e-18, 1e-20, 1e-25, 1e-30, 1e3])[:, None]
    for dtype in (F32, BF16):
        x = (torch.randn(6, K, generator=g) * size).to(dtype)
        w = (1 + 0.2 * torch.randn(K, generator=g)).to(dtype)
        # (eps as the kernel gets it: an fp32 number)
        _, z = exact(x, w, None, float(torch.tensor(eps)), rot)
        check(icq.rms_norm_quantize(x.to(gpu_dev), w.to(gpu_dev), eps=eps, rot_size=rot)[0], z)


def test_one_large_value(gpu_dev):
    """A single value whose square overflows among ordinary ones, and Inf or NaN beside such values."""
    import int_crush_converter_amd as icq
    g = torch.Generator().manual_seed(1)
    for K in (200, 5000, 30000):
        x = torch.randn(4, K, generator=g)
        x[0, 3], x[1, K - 1], x[2, 7], x[3, 9] = 3e38, -1e25, 1e25, -3e38
        x[2, 8], x[3, 10] = float("inf"), float("nan")
        q = icq.rms_norm_quantize(x.to(gpu_dev), torch.ones(K, device=gpu_dev))[0]
        assert torch.isnan(q.scales[2:]).all() and not q.codes[2:].any()
        _, z = exact(x[:2], torch.ones(K), None, 1e-6, 1)
        s = z.abs().amax(1) / 127
        assert ((q.scales[:2].cpu().double() - s).abs() <= 2.0 ** -16 * s).all()
        assert q.codes[0, 3] == 127 and q.codes[1, K - 1] == -127 and int(q.codes[:2].ne(0).sum()) == 2


def test_fp16_rows_are_never_out_of_range(gpu_dev):
    import int_crush_converter_amd as icq
    x = torch.full((3, 65536), 65504.0, dtype=F16)
    x[1] = 2.0 ** -24
    _, z = exact(x, torch.ones(65536, dtype=F16), None, 1e-6, 1)
    check(icq.rms_norm_quantize(x.to(gpu_dev), torch.ones(65536, device=gpu_dev, dtype=F16))[0], z)


@pytest.mark.parametrize("K", [3, 5000, 20000])
def test_the_largest_value_comes_back_finite(gpu_dev, K):
    """The scale of a row that holds fp32's largest value (a mask's, say) gives no infinity when it is undone."""
    import int_crush_converter_amd as icq
    top = torch.finfo(F32).max
    x = torch.randn(4, K)
    x[0, 1], x[1, K - 1], x[2, 0] = top, -top, float(torch.nextafter(torch.tensor(top), torch.tensor(0.0)))
    q = icq.quantize_activations(x.to(gpu_dev))
    check(q, x.double())
    back = q.dequantize(F32).cpu()
    assert torch.isfinite(back).all()
    assert (back[0, 1] / top - 1).abs() < 2.0 ** -22 and (back[1, K - 1] / -top - 1).abs() < 2.0 ** -22
