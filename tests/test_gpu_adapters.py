"""quantized_linear with low-rank adapters against the definition in 64 bits.

Bounds.  y = base + d with d = scaling sum_r b_r t_r, t_r = sum_k a_rk (sa q_k).
Base: 2^-21 of its magnitude (test_gpu_quantized_linear.py).  t: the products of
two 16-bit values and the additions over K in fp32, rounded or truncated, are
within (K + 8) 2^-23 of S_r = sum_k |a_rk q_k sa scaling|, the scalings included.
d: t as two bfloat16 values is within 2^-16 of it (hi truncated, the rest within
2^-7 and rounded to 2^-9 of it), float16 values of b are two bfloat16 values
exactly; the sum over the (padded) rank, both parts and planes within (4 rank +
160) 2^-23 of sum_r |b_r| S_r.  A 16-bit result adds half a step: that
of its type's relative to the value, and below float16's smallest normal number
2^-14, where steps are 2^-24 whatever the value, 2^-25.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
STEP = {F32: 0.0, BF16: 2.0 ** -8, F16: 2.0 ** -11}
SUBNORMAL = {F32: 0.0, BF16: 0.0, F16: 2.0 ** -25}


def pack4(q):
    u = torch.nn.functional.pad(q, (0, q.shape[1] % 2)).view(torch.uint8) & 15
    return u[:, 0::2] | (u[:, 1::2] << 4)


class Case:
    def __init__(self, dev, M, N, K, L, R, bits, asym, dtype, seed, size=1.0):
        import int_crush_converter_amd as icq
        g = torch.Generator().manual_seed(seed)
        lo, hi = (-8, 8) if bits == 4 else (-128, 128)
        self.g, self.dev, self.L = g, dev, L
        self.codes = torch.randint(-128, 128, (M, K), generator=g).to(torch.int8)
        self.sa = torch.rand(M, generator=g) * 0.01 + 1e-4
        self.q = torch.randint(lo, hi, (N, K), generator=g).to(torch.int8)
        self.z = torch.randint(lo, hi, (N,), generator=g).to(torch.int8) if asym else None
        self.s = (torch.rand(N, generator=g) * 0.01 + 1e-4).to(F16)
        self.a = (torch.randn(L, R, K, generator=g) * size).to(dtype)
        self.b = torch.randn(L, N, R, generator=g).to(dtype)
        self.scaling = torch.rand(L, generator=g) + 0.5
        self.bias = torch.randn(N, generator=g)
        self.act = icq.QuantizedActivations.from_codes(self.codes.to(dev), self.sa.to(dev))
        self.w = icq.QuantizedWeight((pack4(self.q) if bits == 4 else self.q).to(dev), self.s.to(dev),
                                     None if self.z is None else self.z.to(dev), in_features=K)
        self.ad = icq.LowRankAdapters(self.a.to(dev), self.b.to(dev), self.scaling.to(dev))

    def run(self, ids, bias=None, out_dtype=F32):
        import int_crush_converter_amd as icq
        return icq.quantized_linear(self.act, self.w, None if bias is None else bias.to(self.dev), adapters=self.ad,
                                    groups=icq.group_rows(ids.to(self.dev), self.L), out_dtype=out_dtype)

    def check(self, y, ids, bias=None):
        x = self.codes.double() * self.sa.double()[:, None]
        w = self.q.double() - (0 if self.z is None else self.z.double()[:, None])
        want = (x @ w.T) * self.s.double()
        room = want.abs() * 2.0 ** -21
        if bias is not None:
            want = want + bias.double()
            room = room + bias.double().abs() * 2.0 ** -21
        K, R = self.a.shape[2], self.a.shape[1]
        for n in range(self.L):
            at = (ids == n).nonzero()[:, 0]
            if at.shape[0]:
                a, b, s = self.a[n].double(), self.b[n].double(), self.scaling[n].double()
                t, size = s * (x[at] @ a.T), s * (x[at].abs() @ a.abs().T)
                want[at] += t @ b.T
                room[at] += (size @ b.abs().T) * ((K + 8) * 2.0 ** -23 + (4 * R + 160) * 2.0 ** -23) + (t.abs() @ b.abs().T) * 2.0 ** -16
                room[at] += (t @ b.T).abs() * 2.0 ** -22
        got = y.cpu().double()
        assert tuple(got.shape) == tuple(want.shape)
        assert ((got - want).abs() <= room + (want.abs() + room) * STEP[y.dtype] + SUBNORMAL[y.dtype] + 1e-12).all()


SIZES = [  # M, N, K, adapters, rank
    (1, 1, 1, 1, 1), (1, 16, 128, 3, 16), (2, 17, 127, 2, 4), (15, 100, 2, 5, 12), (16, 64, 129, 64, 16), (17, 257, 1000, 9, 64),
    (33, 48, 2901, 1000, 8), (64, 512, 256, 40, 16), (65, 300, 640, 2, 128), (300, 1000, 512, 7, 33), (1, 4096, 4096, 4, 16),
    (700, 1500, 65, 3, 16), (1100, 1000, 300, 30, 24), (2100, 2100, 260, 5, 64), (4200, 2304, 130, 300, 16), (2050, 4100, 64, 2, 128),
    (2050, 4100, 300, 3, 128), (2050, 4100, 4200, 3, 16), (2050, 4104, 4100, 40, 64), (1500, 1400, 193, 1000, 40), (900, 2000, 260, 70, 8), (4100, 2600, 520, 1, 16),
    (70, 7000, 300, 3, 12), (40, 10111, 200, 5, 40), (9, 8200, 260, 4, 16),     # 64 rows x 64 and x 48 columns, 16 x 32
]


@pytest.mark.parametrize("M,N,K,L,R", SIZES)
@pytest.mark.parametrize("dtype,bits,asym", [(BF16, 4, True), (F16, 8, True), (BF16, 8, False), (F16, 4, False)])
def test_against_64_bits(gpu_dev, M, N, K, L, R, dtype, bits, asym):
    c = Case(gpu_dev, M, N, K, L, R, bits, asym, dtype, M + N + K)
    ids = torch.randint(-1, L, (M,), generator=c.g)
    c.check(c.run(ids), ids)
    ids = torch.sort(ids).values                                   # requests' rows one after another
    c.check(c.run(ids, c.bias, dtype), ids, c.bias)


@pytest.mark.parametrize("R", [3, 8, 16, 24, 32, 40, 64, 100, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_rows_that_share_adapters(gpu_dev, R, dtype):
    """Few rows, from one adapter for all 16 of a tile to one for each, one after another and mixed, some with none."""
    for M, N, L in ((3, 37, 2), (16, 200, 16), (33, 130, 5), (50, 3300, 9), (120, 68, 33)):
        c = Case(gpu_dev, M, N, 150, L, R, 4, True, dtype, M + R)
        for of in (1, 2, 4, L):                                   # so many adapters, of which neighbours are seldom the same
            ids = torch.arange(M) % min(of, L)
            c.check(c.run(ids), ids)
            ids[torch.rand(M, generator=c.g) < 0.2] = -1
            c.check(c.run(ids), ids)
            ids = (torch.arange(M) * of // M).clamp(max=L - 1)    # and one after another
            c.check(c.run(ids), ids)


def test_sizes_reach_every_form(gpu_dev):
    """Tiles of 256 x 256 need K = 4096 here."""
    import int_crush_converter_amd._native as nat
    assert {(nat.lib().ic_linear_form(k, m, n), d >= 4096) for m, n, d, _, _ in SIZES for k in (0, 1)} >= {(0, False), (0, True), (128, False), (256, False), (256, True)}


@pytest.mark.parametrize("M,N", [(40, 60), (1500, 1400), (2500, 4096)])
def test_rows_without_adapter_have_the_plain_products_bits(gpu_dev, M, N):
    import int_crush_converter_amd as icq
    c = Case(gpu_dev, M, N, 200, 4, 16, 4, True, BF16, M)
    for out in (F32, BF16, F16):
        plain = icq.quantized_linear(c.act, c.w, c.bias.to(gpu_dev), out_dtype=out)
        none = torch.full((M,), -1)
        assert torch.equal(c.run(none, c.bias, out), plain)
        assert torch.equal(c.run(torch.full((M,), 99), c.bias, out), plain)
        ids = torch.randint(-1, 4, (M,), generator=c.g)
        y = c.run(ids, c.bias, out)
        assert torch.equal(y[(ids < 0).to(gpu_dev)], plain[(ids < 0).to(gpu_dev)])
        assert not torch.equal(y, plain)


@pytest.mark.parametrize("M,N", [(40, 60), (1500, 1400), (2500, 4100)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_an_adapter_reaches_its_own_rows_only(gpu_dev, M, N, dtype):
    """Inf and NaN in one adapter's first factor, and in one row's scale, stay there."""
    import int_crush_converter_amd as icq
    c = Case(gpu_dev, M, N, 130, 3, 20, 8, True, dtype, M)
    ids = torch.randint(-1, 3, (M,), generator=c.g)
    y = c.run(ids)
    bad = c.a.clone()
    bad[1, 3, 5] = float("nan")
    bad[1, 7, 2] = float("inf")
    got = icq.quantized_linear(c.act, c.w, adapters=icq.LowRankAdapters(bad, c.b, c.scaling),
                               groups=icq.group_rows(ids.to(gpu_dev), 3), out_dtype=F32)
    mine = (ids == 1).to(gpu_dev)
    assert torch.equal(got[~mine], y[~mine])
    assert not torch.isfinite(got[mine]).any()
    sa = c.sa.clone()
    sa[M // 2] = float("nan")
    act = icq.QuantizedActivations.from_codes(c.codes.to(gpu_dev), sa.to(gpu_dev))
    got = icq.quantized_linear(act, c.w, adapters=c.ad, groups=icq.group_rows(ids.to(gpu_dev), 3), out_dtype=F32)
    assert torch.isnan(got[M // 2]).all()
    got[M // 2] = y[M // 2]
    assert torch.equal(got, y)


@pytest.mark.parametrize("M,N", [(20, 64), (1500, 1400)])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("size,scale", [(1.0, 1e12), (1.0, 1e-30), (1e-3, 1e-12)])
def test_the_adapters_range(gpu_dev, M, N, dtype, size, scale):
    """t far outside 16 bits' range: the row's magnitude is no matter."""
    import int_crush_converter_amd as icq
    c = Case(gpu_dev, M, N, 200, 2, 16, 8, False, dtype, M, size)
    c.scaling = c.scaling * scale
    c.ad = icq.LowRankAdapters(c.a, c.b, c.scaling)
    ids = torch.randint(-1, 2, (M,), generator=c.g)
    c.check(c.run(ids), ids)


def test_lead_shapes_strides_and_scalings(gpu_dev):
    import int_crush_converter_amd as icq
    g = torch.Generator().manual_seed(2)
    K, N, L, R = 256, 96, 3, 8
    w = icq.QuantizedWeight(torch.randint(-128, 128, (N, K), generator=g).to(torch.int8).to(gpu_dev), torch.full((N,), 0.01, device=gpu_dev))
    a, b = torch.randn(L, R, K, generator=g).to(BF16).to(gpu_dev), torch.randn(L, N, R, generator=g).to(BF16).to(gpu_dev)
    act = icq.quantize_activations(torch.randn(2, 5, K, generator=g).to(gpu_dev))
    ids = torch.randint(0, L, (2, 5), generator=g).to(gpu_dev)
    groups = icq.group_rows(ids.reshape(-1), L)
    y = icq.quantized_linear(act, w, adapters=icq.LowRankAdapters(a, b, 2.0), groups=groups)
    assert tuple(y.shape) == (2, 5, N)
    turned = icq.LowRankAdapters(a.transpose(1, 2).contiguous().transpose(1, 2), b.transpose(0, 2).contiguous().transpose(0, 2),
                                 torch.tensor([2.0], dtype=torch.float64))
    assert torch.equal(icq.quantized_linear(act, w, adapters=turned, groups=groups), y)
    host = icq.LowRankAdapters(a.cpu(), b.cpu(), torch.full((L,), 2.0))
    assert torch.equal(icq.quantized_linear(act, w, adapters=host, groups=groups), y)
    none = icq.QuantizedActivations.from_codes(torch.zeros(0, K, dtype=torch.int8, device=gpu_dev), torch.zeros(0, device=gpu_dev))
    empty = icq.quantized_linear(none, w, adapters=host, groups=icq.group_rows(torch.zeros(0, dtype=torch.int32, device=gpu_dev), L))
    assert tuple(empty.shape) == (0, N)


def test_rotated_layers(gpu_dev):
    """Beside a rotated weight the adapter's first factor is rotated like it: the same adapter in the end.  Rotation and
    its rounding to bfloat16 move t by 2^-8 of sum |a x| at most twice, the 8-bit activations are the same."""
    import int_crush_converter_amd as icq
    g = torch.Generator().manual_seed(5)
    K, N, R, rot = 200, 48, 8, 64
    x = torch.randn(30, K, generator=g)
    a, b = torch.randn(1, R, K, generator=g), torch.randn(1, N, R, generator=g)
    act = icq.quantize_activations(x.to(gpu_dev), rot_size=rot)
    Kp = act.in_features
    w = icq.QuantizedWeight(torch.zeros(N, Kp, dtype=torch.int8, device=gpu_dev), torch.ones(N, device=gpu_dev))
    turned = icq.rotate_weights(a[0].to(gpu_dev), rot)[None].to(BF16)
    assert tuple(turned.shape) == (1, R, Kp)
    ad = icq.LowRankAdapters(turned, b.to(BF16), 1.0)
    y = icq.quantized_linear(act, w, adapters=ad, groups=icq.group_rows(torch.zeros(30, dtype=torch.int32), 1), out_dtype=F32)
    back = act.dequantize(F32).cpu().double()                      # R x as its codes say
    exact = back @ turned[0].cpu().double().T @ b[0].to(BF16).double().T
    room = back.abs() @ turned[0].cpu().double().abs().T @ b[0].to(BF16).double().abs().T
    assert ((y.cpu().double() - exact).abs() <= room * ((2 * Kp + 200) * 2.0 ** -23 + 2.0 ** -16)).all()
    straight = x.double() @ a[0].double().T @ b[0].double().T
    # codes are within half a step of R x, a step being the row's largest / 127, and each |R a| within 2^-8 of itself, b too
    step = act.scales.cpu().double()[:, None] / 2
    off = (step * turned[0].cpu().double().abs().sum(1)) @ b[0].double().abs().T + room * 2.0 ** -6
    assert ((y.cpu().double() - straight).abs() <= off).all()


def test_other_stream_and_graph(gpu_dev):
    import int_crush_converter_amd as icq
    for M, N in ((9, 60), (1500, 1400)):
        c = Case(gpu_dev, M, N, 200, 5, 16, 4, True, BF16, M)
        ids = torch.randint(-1, 5, (M,), generator=c.g).to(gpu_dev)
        x = torch.randn(M, 200, generator=c.g).to(gpu_dev)

        def chain():
            act = icq.quantize_activations(x)
            groups = icq.group_rows(ids, 5)
            return icq.quantized_linear(act, c.w, adapters=c.ad, groups=groups), icq.quantized_linear(act, c.w, c.bias.to(gpu_dev).to(BF16), adapters=c.ad, groups=groups)

        c.bias = c.bias.to(gpu_dev)
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
            x.copy_(torch.randn(M, 200, generator=c.g))
            ids.copy_(torch.randint(-1, 5, (M,), generator=c.g))
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in held]
            assert all(torch.equal(a, b) for a, b in zip(got, chain())), k
