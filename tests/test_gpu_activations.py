"""8-bit activations (rms_norm_quantize, quantize_activations) against a
64-bit restatement.

Bounds.  Of a group of 256 values the rotation forms sums over 4 stages of 4
terms: its error is at most 12 2^-24 sum|y| / 16 <= 12 2^-24 |z|_2 <= 12 2^-24
16 max|z|; the norm's own few roundings (2^-22 a value) pass through the same
factor 16.  Together under 2^-16 of the row's maximum, so a code is within
0.5 + 127 * 2^-16 of the exact quotient and a scale within 2^-16 of its value.
"""

from __future__ import annotations

import pytest
import torch

from oracle import torch_ref as ref

pytestmark = pytest.mark.gpu

REL = 2.0 ** -16
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def exact(x, weight, residual, eps, rot):
    h = x.double() if residual is None else x.double() + residual.double()
    y = h
    if weight is not None:
        y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * weight.double()
    if rot > 1:
        y = torch.nn.functional.pad(y, (0, -y.shape[-1] % rot))
        H = ref.hadamard_regular(rot, torch.float64)
        y = (y.reshape(-1, rot) @ H.T).reshape(*x.shape[:-1], -1)
    return h, y


def check(q, z):
    z = z.reshape(-1, z.shape[-1])
    s = z.abs().amax(1).clamp(min=1e-30) / 127
    assert q.in_features == z.shape[1]
    codes = q.codes.reshape(-1, z.shape[1]).cpu()
    got = q.scales.cpu().double()
    assert ((got - s).abs() <= REL * s).all()
    off = (codes.double() - z / s[:, None]).abs().max().item() if z.numel() else 0.0
    assert off <= 0.5 + 127 * REL, off
    assert torch.equal(q.sums.cpu().long(), codes.long().sum(1))
    assert not q.data[:, z.shape[1]:].any()
    for dt in (BF16, F32):
        want = (codes.float() * q.scales.cpu()[:, None]).to(dt)
        assert torch.equal(q.dequantize(dt).reshape(-1, z.shape[1]).cpu(), want)


CASES = [(1, 1, 0, F32), (1, 16, 16, BF16), (3, 17, 16, F16), (2, 255, 256, F32), (5, 1024, 0, BF16), (4, 1025, 64, F16),
         (9, 1040, 4, BF16), (7, 4096, 256, BF16), (3, 4112, 0, F32), (2, 12288, 256, F16), (2, 16385, 64, BF16),
         (1, 65536, 256, F32), (1, 2901, 256, F16), (130, 2048, 256, BF16), (33, 5000, 16, F16), (600, 640, 64, BF16)]


@pytest.mark.parametrize("rows,K,rot,dtype", CASES)
@pytest.mark.parametrize("norm,residual", [(True, True), (True, False), (False, False)])
def test_against_64_bits(gpu_dev, rows, K, rot, dtype, norm, residual):
    import int_crush_converter_amd as icq
    g = torch.Generator().manual_seed(rows * 7919 + K)
    x = (torch.randn(rows, K, generator=g) * torch.where(torch.rand(K, generator=g) < 0.02, 12.0, 1.0)).to(dtype)
    r = (torch.randn(rows, K, generator=g) * 3).to(dtype) if residual else None
    w = (1 + 0.2 * torch.randn(K, generator=g)).to(dtype) if norm else None
    h, z = exact(x, w, r, 1e-6, rot)
    if norm:
        q, out = icq.rms_norm_quantize(x.to(gpu_dev), w.to(gpu_dev), None if r is None else r.to(gpu_dev), eps=1e-6,
                                       rot_size=rot)
        if residual:
            assert torch.equal(out.cpu(), (x.float() + r.float()).to(dtype))
        else:
            assert out is None
    else:
        q = icq.quantize_activations(x.to(gpu_dev), rot_size=rot)
    check(q, z)


def test_shapes_strides_and_weight_types(gpu_dev):
    import int_crush_converter_amd as icq
    g = torch.Generator().manual_seed(3)
    base = torch.randn(6, 10, 700, generator=g)
    for x in (base, base[:, ::2, :640], base[:, :, 3:515], base.transpose(1, 2), base[0, :, 1::2],
              base[:1].expand(4, 10, 700), base[0, 0]):
        K = x.shape[-1]
        w = 1 + 0.1 * torch.randn(K, generator=g)
        for dt, wt in ((F32, F32), (BF16, F32), (F16, BF16)):
            xs, ws = x.to(dt), w.to(wt)
            xg = x.to(gpu_dev).to(dt)                            # .to keeps the strides
            q, out = icq.rms_norm_quantize(xg, ws.to(gpu_dev), xg, rot_size=16)
            h, z = exact(xs, ws, xs, 1e-6, 16)
            assert q.codes.shape == (*x.shape[:-1], q.in_features)
            assert torch.equal(out.cpu(), (xs.float() + xs.float()).to(dt))
            check(q, z)
    pitched = torch.randn(5, 1000, generator=g).to(gpu_dev)[:, 8:520]     # rows at a pitch, aligned
    check(icq.quantize_activations(pitched), pitched.cpu().double())
    odd = torch.randn(5, 1001, generator=g).to(gpu_dev)[:, 1:513]         # a pitch that is not aligned
    check(icq.quantize_activations(odd), odd.cpu().double())


def test_empty_zero_and_tiny_rows(gpu_dev):
    import int_crush_converter_amd as icq
    for shape in ((0, 64), (2, 0, 64)):
        q, out = icq.rms_norm_quantize(torch.empty(shape, device=gpu_dev), torch.ones(64, device=gpu_dev),
                                       torch.empty(shape, device=gpu_dev), rot_size=64)
        assert q.codes.shape == shape and out.shape == shape and q.dequantize().shape == shape
    x = torch.zeros(4, 300)
    x[1] = 1e-38 * torch.randn(300)
    x[2, 7] = 65504.0
    x[3, 299] = -3e38
    q = icq.quantize_activations(x.to(gpu_dev))
    assert not q.codes[0].any() and q.sums[0] == 0 and torch.isfinite(q.scales).all()
    assert not q.codes[1].any()                              # below 1e-30: nothing is left
    assert q.codes[2, 7] == 127 and q.codes[3, 299] == -127
    assert torch.equal(q.dequantize(F32).cpu()[0], torch.zeros(300))


@pytest.mark.parametrize("rows", [1, 5])
@pytest.mark.parametrize("K", [64, 2048, 5120, 20480])
def test_nonfinite_rows_stay_alone(gpu_dev, rows, K):
    import int_crush_converter_amd as icq
    g = torch.Generator().manual_seed(K)
    for bad in (float("nan"), float("inf"), -float("inf")):
        x = torch.randn(rows + 2, K, generator=g)
        clean = x.clone()
        x[1, K // 3] = bad
        for norm in (False, True):
            w = torch.ones(K, device=gpu_dev)
            f = (lambda t: icq.rms_norm_quantize(t, w, rot_size=64)[0]) if norm else icq.quantize_activations
            q, c = f(x.to(gpu_dev)), f(clean.to(gpu_dev))
            assert torch.isnan(q.scales[1]) and not q.codes[1].any() and q.sums[1] == 0
            assert torch.isnan(q.dequantize()[1]).all()
            keep = [i for i in range(rows + 2) if i != 1]
            assert torch.equal(q.codes[keep], c.codes[keep]) and torch.equal(q.scales[keep], c.scales[keep])


def test_from_codes(gpu_dev):
    import int_crush_converter_amd as icq
    g = torch.Generator().manual_seed(9)
    for rows, K in ((1, 1), (3, 127), (4, 128), (5, 1000), (0, 256)):
        c = torch.randint(-128, 128, (rows, K), generator=g).to(torch.int8)
        s = torch.rand(rows, generator=g)
        q = icq.QuantizedActivations.from_codes(c.to(gpu_dev), s.to(gpu_dev))
        assert torch.equal(q.codes.cpu(), c) and torch.equal(q.sums.cpu().long(), c.long().sum(1))
        assert torch.equal(q.dequantize(F32).cpu(), c.float() * s[:, None])
    c = torch.randint(-128, 128, (6, 256), generator=g).to(torch.int8).to(gpu_dev)
    q = icq.QuantizedActivations.from_codes(c[:, :128], torch.ones(6, device=gpu_dev))     # a slice is copied
    assert torch.equal(q.codes, c[:, :128])
    assert torch.equal(q.sums.long(), c[:, :128].long().sum(1))


def test_refusals(gpu_dev):
    import int_crush_converter_amd as icq
    x, w = torch.randn(4, 64, device=gpu_dev), torch.ones(64, device=gpu_dev)
    for rot in (2, 3, 32, 128, 512, -1):
        with pytest.raises(ValueError, match="rot_size"):
            icq.quantize_activations(x, rot_size=rot)
    with pytest.raises(ValueError, match="weight"):
        icq.rms_norm_quantize(x, torch.ones(63, device=gpu_dev))
    with pytest.raises(ValueError, match="weight"):
        icq.rms_norm_quantize(x, None)
    with pytest.raises(ValueError, match="residual"):
        icq.rms_norm_quantize(x, w, x[:3])
    with pytest.raises(ValueError, match="residual"):
        icq.rms_norm_quantize(x, w, x.half())
    with pytest.raises(TypeError):
        icq.quantize_activations(x.double())
    with pytest.raises(ValueError, match="in_features"):
        icq.quantize_activations(torch.empty(2, 65537, device=gpu_dev))
    with pytest.raises(ValueError, match="in_features"):
        icq.quantize_activations(torch.empty(2, 0, device=gpu_dev))
    with pytest.raises(ValueError, match="int8"):
        icq.QuantizedActivations.from_codes(x, torch.ones(4, device=gpu_dev))
    with pytest.raises(ValueError, match="scales"):
        icq.QuantizedActivations.from_codes(x.to(torch.int8), torch.ones(3, device=gpu_dev))
