"""The products' tiled forms, at sizes that the form's rule sends there
(ic_linear_form is asked, so that a changed rule does not leave them untested):
tiles that end inside the matrix, more tiles than work-groups, rows of the
output at any alignment, K of fewer stages than there are buffers and of more.

Bounds.  The integer sums are exact: fp32 results are within 2^-21 of |y| +
|bias| (four roundings, doubled for the intermediate values).  Products of two
E2M1 values with their scales are exact in fp32 and a sum of K of them in any
order within (K + 8) 2^-23 sum|a w|; the bias adds one rounding.  16-bit results
are the fp32 results rounded once, bit for bit.
"""

from __future__ import annotations

import os

import pytest
import torch

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
KINDS = [(8, True), (8, False), (4, True), (4, False), ("mx", False)]
# form, M, N: one tile row short, rows of y at no alignment, few rows and many columns; more than one tile a work-group
SIZES = [(128, 1345, 1000), (128, 1345, 1003), (128, 65, 16000), (128, 4400, 3704), (128, 4400, 3701),
         (256, 3300, 3904), (256, 3300, 3901), (256, 5100, 5104), (256, 5100, 5101)]
DEPTHS = [1, 65, 129, 250, 257, 385, 513, 2901]


def form(kind, M, N):
    from int_crush_converter_amd import _native as nat
    nat.load(require_gpu=False)
    return nat._lib.ic_linear_form({8: 0, 4: 1, "mx": 2}[kind], M, N)


def test_sizes_reach_the_forms():
    from int_crush_converter_amd import _native as nat
    if not os.path.exists(nat.LIB_PATH):
        from int_crush_converter_amd import build
        build.build()
    assert all(form(kind, M, N) == f for f, M, N in SIZES for kind in (4, 8, "mx"))
    assert form(4, 1, 1 << 20) == 0 and form(8, 64, 1 << 20) == 0 and form("mx", 0, 5) == 0
    # the lines: work-groups of the direct form; half of a round of 256 tiles, three quarters (INT4: two thirds) of several
    assert [form(k, m, 4096) for k in (8, 4, "mx") for m in (192, 256, 320, 384)] == [0, 128, 128, 128, 0, 0, 0, 128, 0, 0, 128, 128]
    assert [form(8, m, 4096) for m in (2048, 2049, 4096, 4097, 5888, 5889)] == [128, 256, 256, 128, 128, 256]
    assert [form(4, m, 4096) for m in (2048, 2049, 4096, 4097, 5376, 5377)] == [128, 256, 256, 128, 128, 256]
    form(8, 1, 1)
    L = nat._lib.ic_linear_form
    assert L(0, -1, 5) == -1 and L(0, 5, 0) == -1 and L(3, 5, 5) == -1 and L(-1, 5, 5) == -1


class Problem:
    """Operands on the GPU, the product in 64 bits and the room that an fp32 result has."""

    def __init__(self, kind, asym, M, N, K, dev, seed, with_bias=True):
        import int_crush_converter_amd as icq
        self.kind, self.K = kind, K
        g = torch.Generator(device=dev).manual_seed(seed)
        ints = lambda lo, hi, *size: torch.randint(lo, hi, size, generator=g, device=dev)      # noqa: E731
        self.bias = torch.randn(N, generator=g, device=dev) if with_bias else None
        b64 = 0 if self.bias is None else self.bias.double()
        if kind == "mx":
            grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64, device=dev)

            def operand(rows):
                codes = ints(0, 256, rows, (K + 1) // 2).to(torch.uint8)
                scales = ints(118, 134, rows, -(-K // 32)).to(torch.uint8)
                v = grid[torch.stack((codes & 15, codes >> 4), 2).reshape(rows, -1)[:, :K].long()]
                return codes, scales, v * torch.exp2(scales.double() - 127).repeat_interleave(32, 1)[:, :K]
            (self.a, self.sa, a64), (self.q, self.sw, w64) = operand(M), operand(N)
            self.want = a64 @ w64.T + b64
            self.room = (K + 8) * 2.0 ** -23 * (a64.abs() @ w64.abs().T) + 2.0 ** -23 * self.want.abs()
            self.w = icq.Mxfp4Tensor.from_packed(self.q, self.sw, in_features=K)
        else:
            lo, hi = (-8, 8) if kind == 4 else (-128, 128)
            self.a, self.sa = ints(-128, 128, M, K).to(torch.int8), torch.rand(M, generator=g, device=dev) * 0.01 + 1e-4
            q = ints(lo, hi, N, K).to(torch.int8)
            z = ints(lo, hi, N, 1).to(torch.int8) if asym else None
            sw = (torch.rand(N, 1, generator=g, device=dev) * 0.01 + 1e-4).half()
            if kind == 4:
                u = torch.nn.functional.pad(q, (0, K % 2)).view(torch.uint8) & 15
                stored = u[:, 0::2] | (u[:, 1::2] << 4)
            self.w = icq.QuantizedWeight(stored if kind == 4 else q, sw, z, in_features=K)
            w64 = q.double() - (0 if z is None else z.double())
            self.want = (self.a.double() @ w64.T) * self.sa.double()[:, None] * sw.double().reshape(1, -1) + b64
            self.room = 2.0 ** -21 * (self.want.abs() + (0 if self.bias is None else self.bias.abs().double())) + 1e-12

    def activations(self, rows=slice(None)):
        import int_crush_converter_amd as icq
        if self.kind == "mx":
            return icq.Mxfp4Tensor.from_packed(self.a[rows], self.sa[rows], in_features=self.K)
        return icq.QuantizedActivations.from_codes(self.a[rows], self.sa[rows])

    def run(self, act, dtype=F32):
        import int_crush_converter_amd as icq
        f = icq.mxfp4_linear if self.kind == "mx" else icq.quantized_linear
        return f(act, self.w, self.bias, out_dtype=dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,asym", KINDS)
@pytest.mark.parametrize("tile,M,N", SIZES)
def test_against_64_bits(gpu_dev, tile, M, N, kind, asym):
    assert form(kind, M, N) == tile
    for K in DEPTHS:
        p = Problem(kind, asym, M, N, K, gpu_dev, M + N + K, with_bias=K % 2 == 1)
        act = p.activations()
        y = p.run(act)
        bad = (y.double() - p.want).abs() > p.room
        assert y.shape == (M, N) and not bad.any(), (K, int(bad.sum()), bad.nonzero()[:4].tolist())
        for dt in (BF16, F16):
            assert torch.equal(p.run(act, dt), y.to(dt)), (K, dt)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,asym", KINDS)
def test_rows_do_not_depend_on_the_form(gpu_dev, kind, asym):
    """Rows of a batch by tiles of 256 against the same rows by tiles of 128 and directly: equal where the sums are
    exact, within both results' room in E2M1."""
    M, N, K = 3300, 3901, 1300
    p = Problem(kind, asym, M, N, K, gpu_dev, 11)
    full = p.run(p.activations())
    seen = {form(kind, M, N)}
    for lo, hi in ((0, 1500), (700, 2000), (100, 165), (3299, 3300), (256, 320), (1, 18)):
        seen.add(form(kind, hi - lo, N))
        part = p.run(p.activations(slice(lo, hi)))
        if kind == "mx":
            assert ((part.double() - full[lo:hi].double()).abs() <= 2 * p.room[lo:hi]).all()
        else:
            assert torch.equal(part, full[lo:hi])
    assert seen == {0, 128, 256}


@pytest.mark.gpu
@pytest.mark.parametrize("tile,M,N", [(128, 1345, 1000), (256, 3300, 3904)])
@pytest.mark.parametrize("bits", [4, 8])
def test_largest_sums(gpu_dev, bits, tile, M, N):
    """Codes at the ends of their ranges over the longest K: the 32-bit sums and the 24-bit zero-point products hold."""
    import int_crush_converter_amd as icq
    assert form(bits, M, N) == tile
    K = 65536
    lo, hi = (-8, 7) if bits == 4 else (-128, 127)
    for qv, zv in ((lo, hi), (hi, lo)):
        stored = torch.full((N, K // 2), (qv & 15) * 17, dtype=torch.uint8, device=gpu_dev) if bits == 4 else \
            torch.full((N, K), qv, dtype=torch.int8, device=gpu_dev)
        w = icq.QuantizedWeight(stored, torch.full((N,), 1e-3, device=gpu_dev),
                                torch.full((N,), zv, dtype=torch.int8, device=gpu_dev))
        for av in (-128, 127):
            act = icq.QuantizedActivations.from_codes(torch.full((M, K), av, dtype=torch.int8, device=gpu_dev),
                                                      torch.full((M,), 1e-4, device=gpu_dev))
            y = icq.quantized_linear(act, w, out_dtype=F32).double()
            s = float(torch.tensor(1e-4).double()) * float(torch.tensor(1e-3).double())
            want = float(av) * (qv - zv) * K * s
            assert ((y - want).abs() <= 2.0 ** -21 * abs(want)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("tile,M,N", [(128, 1345, 1003), (128, 4400, 3704), (256, 5100, 5104)])
@pytest.mark.parametrize("kind", [8, 4, "mx"])
def test_nan_scales_stay_in_their_rows(gpu_dev, tile, M, N, kind):
    """A NaN scale in a tile's first, inner and last row makes those rows NaN and no other (in E2M1 one block does, and a
    weight's block its column)."""
    import int_crush_converter_amd as icq
    assert form(kind, M, N) == tile
    p = Problem(kind, kind != "mx", M, N, 700, gpu_dev, 3, with_bias=False)
    rows, cols = [0, 77, tile, tile + 33, M - 1], [5, N - 1]
    want = torch.zeros(M, N, dtype=torch.bool, device=gpu_dev)
    want[rows] = True
    if kind == "mx":
        for i, r in enumerate(rows):
            p.sa[r, 4 * i + i] = 255
        p.sw[cols[0], 0], p.sw[cols[1], 21] = 255, 255
        p.w = icq.Mxfp4Tensor.from_packed(p.q, p.sw, in_features=700)
        want[:, cols] = True
    else:
        p.sa[rows] = float("nan")
    for dt in (F32, BF16):
        y = p.run(p.activations(), dt)
        assert torch.equal(torch.isnan(y), want)
        if dt == F32:
            assert ((y.double() - p.want).abs() <= p.room)[~want].all()


@pytest.mark.gpu
@pytest.mark.parametrize("tile,M,N", [(128, 1345, 1000), (256, 3300, 3904)])
def test_graph_of_tiles(gpu_dev, tile, M, N):
    """A captured chain with tiled products gives the eager result on every replay, eager work in between."""
    import int_crush_converter_amd as icq
    assert {form(k, M, N) for k in (8, 4, "mx")} == {tile}
    g = torch.Generator(device=gpu_dev).manual_seed(M)
    K = 640
    rand = lambda *s: torch.randn(*s, generator=g, device=gpu_dev)                              # noqa: E731
    w8 = icq.QuantizedWeight((rand(N, K) * 30).clamp(-127, 127).to(torch.int8), torch.full((N,), 0.01, device=gpu_dev))
    w4 = icq.QuantizedWeight((rand(N, K // 2) * 60 + 128).clamp(0, 255).to(torch.uint8), torch.full((N,), 0.1, device=gpu_dev))
    wm = icq.mxfp4_quantize(rand(N, K))
    gain, x = torch.ones(K, device=gpu_dev, dtype=BF16), rand(M, K).to(BF16)

    def chain():
        act, _ = icq.rms_norm_quantize(x, gain, rot_size=64)
        return icq.quantized_linear(act, w8), icq.quantized_linear(act, w4), icq.mxfp4_linear(icq.mxfp4_quantize(x), wm)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = chain()
    for k in range(4):
        x.copy_(rand(M, K).to(BF16))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        assert all(torch.equal(a, b) for a, b in zip(got, chain())), k
