"""quantized_linear against the definition in 64 bits.

Bounds.  The integer sums are exact, so an fp32 result has the roundings of
the sum's conversion, of sa * sw, of their product and of the bias addition:
4 2^-24 of (|y| + |bias|), doubled for the intermediate values: 2^-21.  A
16-bit result is the fp32 result rounded once, bit for bit.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TOL = 2.0 ** -21


def pack4(q):
    u = torch.nn.functional.pad(q, (0, q.shape[1] % 2)).view(torch.uint8) & 15
    return u[:, 0::2] | (u[:, 1::2] << 4)


def make(M, N, K, bits, asym, seed, scale_dtype=F16):
    g = torch.Generator().manual_seed(seed)
    lo, hi = (-8, 8) if bits == 4 else (-128, 128)
    a = torch.randint(-128, 128, (M, K), generator=g).to(torch.int8)
    q = torch.randint(lo, hi, (N, K), generator=g).to(torch.int8)
    z = torch.randint(lo, hi, (N, 1), generator=g).to(torch.int8) if asym else None
    sa = torch.rand(M, generator=g) * 0.01 + 1e-4
    sw = (torch.rand(N, 1, generator=g) * 0.01 + 1e-4).to(scale_dtype)
    bias = torch.randn(N, generator=g)
    return a, sa, q, sw, z, bias


def definition(a, sa, q, sw, z, bias):
    w = q.double() if z is None else q.double() - z.double()
    y = (a.double() @ w.T) * sa.double()[:, None] * sw.double().reshape(1, -1)     # the sum is exact in 64 bits
    return y if bias is None else y + bias.double()


def run(dev, a, sa, q, sw, z, bias, bits, out_dtype=F32):
    import int_crush_converter_amd as icq
    act = icq.QuantizedActivations.from_codes(a.to(dev), sa.to(dev))
    w = icq.QuantizedWeight((pack4(q) if bits == 4 else q).to(dev), sw.to(dev), None if z is None else z.to(dev),
                            in_features=q.shape[1])
    return icq.quantized_linear(act, w, None if bias is None else bias.to(dev), out_dtype=out_dtype)


def check(y, want, bias):
    room = want.abs() + (0 if bias is None else bias.double().abs())
    assert y.dtype == F32 and y.shape == want.shape
    assert ((y.cpu().double() - want).abs() <= TOL * room + 1e-12).all()


SIZES = [(1, 1, 1), (1, 16, 128), (2, 17, 127), (15, 100, 2), (16, 64, 129), (17, 257, 1000), (33, 48, 2901),
         (64, 512, 256), (65, 300, 640), (129, 129, 384), (257, 255, 1153), (300, 1000, 512), (1, 4096, 4096),
         (5, 130, 12288), (512, 640, 1024), (700, 264, 65)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("bits,asym", [(4, True), (4, False), (8, True), (8, False)])
def test_against_64_bits(gpu_dev, M, N, K, bits, asym):
    p = make(M, N, K, bits, asym, M * 31 + N * 17 + K)
    check(run(gpu_dev, *p, bits), definition(*p), p[-1])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M,N,K", [(1, 37, 200), (3, 64, 256), (40, 36, 130), (300, 260, 520), (513, 1000, 300)])
def test_output_types_and_bias(gpu_dev, M, N, K, dtype):
    for bits, asym, with_bias, bdt, sdt in ((4, True, True, F32, F32), (8, False, True, BF16, F16),
                                            (4, False, False, F32, F16), (8, True, True, F16, F32)):
        a, sa, q, sw, z, bias = make(M, N, K, bits, asym, 5 * M + N, sdt)
        bias = bias.to(bdt) if with_bias else None
        y = run(gpu_dev, a, sa, q, sw, z, bias, bits)
        check(y, definition(a, sa, q, sw, z, bias), bias)
        assert torch.equal(run(gpu_dev, a, sa, q, sw, z, bias, bits, dtype), y.to(dtype))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("M", [1, 70, 300])
def test_largest_sums(gpu_dev, bits, M):
    """Codes at the ends of their ranges over the longest K: the 32-bit sums hold."""
    N, K = 33, 65536
    lo, hi = (-8, 7) if bits == 4 else (-128, 127)
    for qv, zv in ((lo, hi), (hi, lo), (lo, lo)):
        for av in (-128, 127):
            a = torch.full((M, K), av, dtype=torch.int8)
            q = torch.full((N, K), qv, dtype=torch.int8)
            z = torch.full((N, 1), zv, dtype=torch.int8)
            sa, sw = torch.full((M,), 1e-4), torch.full((N, 1), 1e-3)
            y = run(gpu_dev, a, sa, q, sw, z, None, bits)
            want = float(av) * (qv - zv) * K * float(sa[0].double()) * float(sw[0].double())
            assert torch.allclose(y.double().cpu(), torch.full((M, N), want, dtype=torch.float64), rtol=2.0 ** -21, atol=0)


def test_rows_of_a_batch_equal_single_rows(gpu_dev):
    """Each row's result does not depend on how many rows go with it."""
    import int_crush_converter_amd as icq
    for bits in (4, 8):
        a, sa, q, sw, z, bias = make(530, 272, 1300, bits, True, bits)
        w = icq.QuantizedWeight((pack4(q) if bits == 4 else q).to(gpu_dev), sw.to(gpu_dev), z.to(gpu_dev), in_features=1300)
        ag, sg = a.to(gpu_dev), sa.to(gpu_dev)
        full = icq.quantized_linear(icq.QuantizedActivations.from_codes(ag, sg), w, out_dtype=F32)
        for lo, hi in ((0, 1), (5, 22), (100, 140), (250, 330), (0, 257), (529, 530)):
            part = icq.quantized_linear(icq.QuantizedActivations.from_codes(ag[lo:hi], sg[lo:hi]), w, out_dtype=F32)
            assert torch.equal(part, full[lo:hi])


def test_converter_layer_end_to_end(gpu_dev):
    """A layer quantised by the converter's own step, run on rotated 8-bit activations, against the same arithmetic
    from its stored tensors."""
    import int_crush_converter_amd as icq
    from int_crush_converter_amd import layer as _layer
    g = torch.Generator().manual_seed(1)
    for bits, asym, rot, N, K in ((4, True, 256, 96, 1000), (8, False, 64, 40, 320), (4, False, 16, 33, 47), (8, True, 0, 64, 130)):
        W = torch.randn(N, K, generator=g) * 0.02
        W_work, _ = _layer.prepare_weights(W.to(gpu_dev), rot)
        codes, s16, z8, packed = _layer.rtn_codes(W_work, bits, asym, None)
        Kp = W_work.shape[1]
        w = icq.QuantizedWeight(codes if bits == 8 else packed, s16, z8, in_features=Kp)
        x = torch.randn(2, 5, K, generator=g).to(BF16).to(gpu_dev)
        q, _ = icq.rms_norm_quantize(x, torch.ones(K, device=gpu_dev, dtype=BF16), rot_size=rot)
        y = icq.quantized_linear(q, w, out_dtype=F32)
        assert y.shape == (2, 5, N)
        want = definition(q.codes.reshape(10, Kp).cpu(), q.scales.cpu(), codes.cpu(), s16.cpu(),
                          None if z8 is None else z8.cpu(), None)
        check(y.reshape(10, N), want, None)
        # and near the layer that was quantised: 4-bit rounding leaves about a tenth, 8-bit a hundredth
        h = x.double().cpu().reshape(10, K)
        ideal = (h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6)) @ W.double().T
        rel = (want - ideal).norm() / ideal.norm()
        assert rel < (0.25 if bits == 4 else 0.03), rel


def test_nan_rows_and_empty(gpu_dev):
    import int_crush_converter_amd as icq
    a, sa, q, sw, z, bias = make(70, 50, 300, 4, True, 2)
    sa[3] = float("nan")
    y = run(gpu_dev, a, sa, q, sw, z, bias, 4)
    assert torch.isnan(y[3]).all() and torch.isfinite(y[:3]).all() and torch.isfinite(y[4:]).all()
    w = icq.QuantizedWeight(q.to(gpu_dev), sw.to(gpu_dev))
    empty = icq.QuantizedActivations.from_codes(torch.empty(0, 4, 300, dtype=torch.int8, device=gpu_dev),
                                                torch.empty(0, 4, device=gpu_dev))
    assert icq.quantized_linear(empty, w).shape == (0, 4, 50)


def test_other_stream_and_graph(gpu_dev):
    """Calls follow the current stream; a captured chain gives the eager result on every replay."""
    import int_crush_converter_amd as icq
    g = torch.Generator().manual_seed(4)
    K, N = 1024, 384
    q = torch.randint(-8, 8, (N, K), generator=g).to(torch.int8)
    w = icq.QuantizedWeight(pack4(q).to(gpu_dev), torch.full((N,), 0.01, device=gpu_dev))
    gain = torch.ones(K, device=gpu_dev, dtype=BF16)
    for rows in (1, 300):
        x = torch.randn(rows, K, generator=g).to(BF16).to(gpu_dev)
        r = torch.randn(rows, K, generator=g).to(BF16).to(gpu_dev)

        def chain():
            act, h = icq.rms_norm_quantize(x, gain, r, rot_size=256)
            mx = icq.mxfp4_quantize(h)
            return icq.quantized_linear(act, w), mx.dequantize(), icq.mxfp4_linear(mx, wm)

        wm = icq.mxfp4_quantize(torch.randn(N, K, generator=g).to(gpu_dev))
        eager = [t.clone() for t in chain()]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = chain()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(other, eager))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = chain()
        for k in range(4):
            x.copy_(torch.randn(rows, K, generator=g).to(BF16))
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in held]
            want = chain()
            assert all(torch.equal(a, b) for a, b in zip(got, want)), k


def test_refusals(gpu_dev):
    import int_crush_converter_amd as icq
    q = torch.zeros(32, 128, dtype=torch.int8, device=gpu_dev)
    s = torch.ones(32, 1, device=gpu_dev)
    w = icq.QuantizedWeight(q, s)
    act = icq.quantize_activations(torch.randn(4, 64, device=gpu_dev))
    with pytest.raises(ValueError, match="features"):
        icq.quantized_linear(act, w)
    act = icq.quantize_activations(torch.randn(4, 128, device=gpu_dev))
    with pytest.raises(ValueError, match="bias"):
        icq.quantized_linear(act, w, torch.ones(31, device=gpu_dev))
    with pytest.raises(TypeError):
        icq.quantized_linear(act, w, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="expected int8"):
        icq.QuantizedWeight(q.float(), s)
    with pytest.raises(ValueError, match="scales"):
        icq.QuantizedWeight(q, torch.ones(32, 2, device=gpu_dev))
    with pytest.raises(ValueError, match="in_features"):
        icq.QuantizedWeight(q, s, in_features=127)
    with pytest.raises(ValueError, match="int8"):
        icq.QuantizedWeight(q, s, s)
