"""Low-rank adapters beside a quantised product, results in fp32: what t = A x is held in, and how small or large it may be
beside the product itself."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


# M, N, K, adapters, rank, adapters in use: 16 x 16, 16 x 32, 32 x 32, 64 x 48 and 64 x 64 outputs a work-group, tiles of 128 x
# 128 and 256 x 256; rows that share adapters and rows that seldom do
EXACT = [(1, 16, 130, 1, 1, 1), (5, 100, 100, 3, 7, 3), (16, 8210, 70, 4, 16, 2), (40, 60, 128, 6, 33, 2), (40, 60, 128, 40, 16, 40), (50, 10000, 40, 40, 8, 40),
         (64, 7000, 40, 3, 64, 3), (64, 14400, 40, 2, 16, 1), (300, 70, 130, 5, 128, 5), (1500, 1400, 200, 3, 16, 3), (1500, 1404, 256, 40, 40, 40),
         (2100, 2300, 260, 2, 128, 2), (4200, 2304, 130, 3, 16, 3), (2050, 4100, 4200, 3, 16, 3), (2050, 4104, 4100, 2, 100, 2)]


@pytest.mark.parametrize("M,N,K,L,R,used", EXACT)
@pytest.mark.parametrize("bits,dtype", [(4, BF16), (8, BF16), (4, F16), (8, F16)])
def test_t_has_all_its_bits(gpu_dev, M, N, K, L, R, used, bits, dtype):
    """Whole numbers throughout: |t| < 2^24 has up to 24 bits, column n takes one of its ranks times 1, -1 or 0.5, and the
    product beside it is a whole number too.  Halves below 2^23 are fp32 values, and so is every partial sum: no bit of
    the result may differ.  The sums over K stay below 2^23: |a| <= 2^23 / (128 K)."""
    import int_crush_converter_amd as icq
    g = torch.Generator().manual_seed(M + N + R)
    top = max(1, min(255, 2 ** 23 // (128 * K)))
    codes = torch.randint(64, 128, (M, K), generator=g).to(torch.int8)    # of one sign, as each rank's: t uses its room
    a = (torch.randint(top // 2, top + 1, (L, R, K), generator=g) * (torch.randint(0, 2, (L, R, 1), generator=g) * 2 - 1)).to(dtype)
    q = (torch.rand(N, K, generator=g) < 16 / K).to(torch.int8)           # some 16 ones a row: the product is small
    rank_of, by = torch.randint(0, R, (L, N), generator=g), torch.tensor([1.0, -1.0, 0.5])[torch.randint(0, 3, (L, N), generator=g)]
    b = torch.zeros(L, N, R).scatter_(2, rank_of[:, :, None], by[:, :, None]).to(dtype)
    ids = torch.randint(-1, used, (M,), generator=g)
    stored = q if bits == 8 else torch.nn.functional.pad(q, (0, K % 2)).view(torch.uint8)
    if bits == 4:
        stored = stored[:, 0::2] | (stored[:, 1::2] << 4)
    w = icq.QuantizedWeight(stored.to(gpu_dev), torch.ones(N, device=gpu_dev), in_features=K)
    act = icq.QuantizedActivations.from_codes(codes.to(gpu_dev), torch.ones(M, device=gpu_dev))
    y = icq.quantized_linear(act, w, adapters=icq.LowRankAdapters(a.to(gpu_dev), b.to(gpu_dev)),
                             groups=icq.group_rows(ids.to(gpu_dev), L), out_dtype=F32)
    want = codes.double() @ q.double().T
    for n in range(used):
        at = (ids == n).nonzero()[:, 0]
        t = codes[at].double() @ a[n].double().T
        assert (t.abs() < 2 ** 23).all()
        want[at] += t[:, rank_of[n]] * by[n].double()
    assert torch.equal(y.cpu().double(), want)


@pytest.mark.parametrize("M,N,K,L,R,used", [c[:2] + (140,) + c[3:] for c in EXACT if c[2] < 4096])
@pytest.mark.parametrize("bits,dtype", [(4, BF16), (8, BF16), (4, F16), (8, F16)])
def test_t_of_sixteen_bit_results(gpu_dev, M, N, K, L, R, used, bits, dtype):
    """t as two bfloat16 values, each the nearest, has whole numbers below 2^17: the first leaves at most 2^8.  The product
    beside it is -t and at most two codes, so that the result is a whole number up to 254, which bfloat16 has too; a t that
    is off by one shows."""
    import int_crush_converter_amd as icq
    g = torch.Generator().manual_seed(M + N + R)
    codes = torch.randint(100, 128, (M, K), generator=g).to(torch.int8)
    rows = torch.randint(5, 8, (R, K), generator=g)                        # t: 140 x 100 x 5 = 2^16.1 to 140 x 127 x 7 < 2^17
    q = -rows[torch.arange(N) % R]
    q[torch.arange(N)[:, None], torch.randint(0, K, (N, 1), generator=g)] += 1
    q[torch.arange(N), torch.randint(0, K, (N,), generator=g)] += 1
    q = q.to(torch.int8)
    place = torch.stack([torch.randperm(R, generator=g) for _ in range(L)])   # adapter l has row r at place[l, r]
    a = torch.zeros(L, R, K).scatter_(1, place[:, :, None].expand(L, R, K), rows.float()[None].expand(L, R, K).contiguous()).to(dtype)
    b = torch.zeros(L, N, R).scatter_(2, place[:, torch.arange(N) % R][:, :, None], 1.0).to(dtype)
    ids = torch.randint(-1, used, (M,), generator=g)
    u = q.view(torch.uint8) & 15
    w = icq.QuantizedWeight((u[:, 0::2] | (u[:, 1::2] << 4) if bits == 4 else q).to(gpu_dev), torch.ones(N, device=gpu_dev), in_features=K)
    act = icq.QuantizedActivations.from_codes(codes.to(gpu_dev), torch.ones(M, device=gpu_dev))
    want = codes.double() @ q.double().T
    t = codes.double() @ rows.double().T
    assert (t < 2 ** 17).all() and (t >= 2 ** 16).all()
    want[ids >= 0] += t[ids >= 0][:, torch.arange(N) % R]
    assert (want[ids >= 0].abs() <= 254).all()
    ad, groups = icq.LowRankAdapters(a.to(gpu_dev), b.to(gpu_dev)), icq.group_rows(ids.to(gpu_dev), L)
    for out in (BF16, F16):
        y = icq.quantized_linear(act, w, adapters=ad, groups=groups, out_dtype=out)
        assert torch.equal(y.cpu(), want.float().to(out))


def test_the_largest_t(gpu_dev):
    """t within 2^-9 of fp32's largest value, whose nearest bfloat16 value is infinite."""
    import int_crush_converter_amd as icq
    K, N = 128, 32
    w = icq.QuantizedWeight(torch.zeros(N, K, dtype=torch.int8, device=gpu_dev), torch.ones(N, device=gpu_dev))
    a, b = torch.zeros(1, 1, K, dtype=BF16), torch.full((1, N, 1), 2.0 ** -40, dtype=BF16)
    a[0, 0, 0] = 1.0
    top = torch.finfo(F32).max
    for scale in (top, -top, top * (1 - 2.0 ** -10), top * (1 - 2.0 ** -8)):
        ad = icq.LowRankAdapters(a.to(gpu_dev), b.to(gpu_dev), scale)
        for M in (3, 700):
            codes = torch.zeros(M, K, dtype=torch.int8)
            codes[:, 0] = 1
            act = icq.QuantizedActivations.from_codes(codes.to(gpu_dev), torch.ones(M, device=gpu_dev))
            groups = icq.group_rows(torch.zeros(M, dtype=torch.int32, device=gpu_dev), 1)
            want = torch.tensor(scale, dtype=F32).double() * 2.0 ** -40
            for out, room in ((F32, 2.0 ** -22), (BF16, 2.0 ** -8 + 2.0 ** -15)):
                y = icq.quantized_linear(act, w, adapters=ad, groups=groups, out_dtype=out)
                assert ((y.cpu().double() - want).abs() <= want.abs() * room).all(), (scale, M, out)


def test_sizes_reach_every_form(gpu_dev):
    import int_crush_converter_amd._native as nat
    assert {(nat.lib().ic_linear_form(k, m, n), d >= 4096) for m, n, d, _, _, _ in EXACT for k in (0, 1)} >= {(0, False), (128, False), (256, False), (256, True)}


class Parts:
    """A product and adapters whose base and added part are known in 64 bits, with the magnitudes of the part's sums."""

    def __init__(self, dev, M, N, K, L, R, bits, dtype, a, b, scaling, weight, seed):
        import int_crush_converter_amd as icq
        g = torch.Generator().manual_seed(seed)
        codes, sa = torch.randint(-128, 128, (M, K), generator=g).to(torch.int8), torch.rand(M, generator=g) * 0.01 + 1e-4
        q = torch.randint(-8, 8, (N, K), generator=g).to(torch.int8) * weight
        a, b = (torch.randn(L, R, K, generator=g) * a).to(dtype), (torch.randn(L, N, R, generator=g) * b).to(dtype)
        s = (torch.rand(L, generator=g) + 0.5) * scaling
        ids = torch.randint(-1, L, (M,), generator=g)
        u = torch.nn.functional.pad(q, (0, K % 2)).view(torch.uint8) & 15
        w = icq.QuantizedWeight((u[:, 0::2] | (u[:, 1::2] << 4) if bits == 4 else q).to(dev), torch.ones(N, device=dev), in_features=K)
        act = icq.QuantizedActivations.from_codes(codes.to(dev), sa.to(dev))
        y = icq.quantized_linear(act, w, adapters=icq.LowRankAdapters(a.to(dev), b.to(dev), s.to(dev)),
                                 groups=icq.group_rows(ids.to(dev), L), out_dtype=F32)
        self.y, x = y.cpu().double(), codes.double() * sa.double()[:, None]
        self.base, self.added, self.room = x @ q.double().T, torch.zeros(M, N, dtype=torch.float64), torch.zeros(M, N, dtype=torch.float64)
        for n in range(L):
            at = (ids == n).nonzero()[:, 0]
            self.added[at] = s[n].double() * (x[at] @ a[n].double().T) @ b[n].double().T
            self.room[at] = s[n].double() * (x[at].abs() @ a[n].double().abs().T) @ b[n].double().abs().T
        # t: K products and some joins and scalings; d: three values of t and two of b for each of the padded ranks, and joins
        self.room *= (K + 8 + 6 * -(-R // 32) * 32 + 200) * 2.0 ** -23


@pytest.mark.parametrize("M,N,K", [(20, 64, 200), (70, 1000, 200), (1500, 1400, 200), (2100, 4000, 4200)])
@pytest.mark.parametrize("bits,dtype,a,b,scaling", [(8, BF16, 1.0, 1.0, 1e-30), (4, F16, 1.0, 1.0, 1e-30), (8, F16, 1e-3, 1.0, 1e-12), (4, BF16, 1e-3, 1.0, 1e-12),
                                                    (4, F16, 1e-6, 1e-6, 1.0), (8, F16, 1e-6, 1e-6, 1e-6), (8, BF16, 1e-20, 1e-6, 1.0), (4, F16, 1.0, 1e3, 1e12)])
def test_small_and_large_adapters_alone(gpu_dev, M, N, K, bits, dtype, a, b, scaling):
    """The weight is of zeros, so that nothing but the adapters' own sums gives room: a part that is lost or flushed to zero
    shows at any magnitude (1e-6 is below float16's normal numbers).  Products below fp32's smallest normal number 2^-126
    count as lost: the values here are above 2^-126 by 2^24 and more, but for those far below their row's others."""
    c = Parts(gpu_dev, M, N, K, 2, 16, bits, dtype, a, b, scaling, 0, M + bits)
    assert (c.base == 0).all() and c.added.abs().max() > 0
    assert ((c.y - c.added).abs() <= c.room).all()
    assert (c.y[c.added == 0] == 0).all()


@pytest.mark.parametrize("M,N,K", [(20, 64, 200), (64, 14400, 136), (1500, 1400, 200), (2100, 4000, 4200)])
@pytest.mark.parametrize("bits,dtype", [(4, BF16), (8, BF16), (4, F16), (8, F16)])
@pytest.mark.parametrize("share", [1e-2, 1e-3])
def test_small_adapters_beside_a_large_product(gpu_dev, M, N, K, bits, dtype, share):
    """The forms for few rows add the adapters' part once.  The tiled ones add it to the value as the matrix instructions go:
    at most one rounding or truncation of the value, 2^-23 of it, for each product: 16 ranks (padded to 32), three values of t
    and a plane of zeros, and as many again for the second plane of float16 factors.  2^-21: the value's own roundings."""
    R = 16
    size = (share / (R * 200) ** 0.5 * 5) ** 0.5                    # base: sqrt(K) 5 sa |q|; part: sqrt(R K) a b sa |q|
    c = Parts(gpu_dev, M, N, K, 2, R, bits, dtype, size, size, 1.0, 1, M)
    planes = 32 * 4 * (1 if dtype == BF16 else 2)
    tiled = M > 100
    value = c.base.abs() + (c.added.abs() + c.room if tiled else 0)
    room = c.room + value * (2.0 ** -21 + (planes * 2.0 ** -23 if tiled else 0)) + c.added.abs() * 2.0 ** -22
    assert ((c.y - c.base - c.added).abs() <= room).all()
    assert (c.added.abs() > 2 * room).any()                        # (a part that is lost would show)


@pytest.mark.parametrize("bits", [4, 8])
def test_as_many_rows_as_there_may_be(gpu_dev, bits):
    """The largest batch and rank, t whole: a workspace of 1 GB, and whole numbers as above."""
    import int_crush_converter_amd as icq
    g = torch.Generator(device=gpu_dev).manual_seed(bits)
    M, N, K, L, R = 1048560, 16, 136, 3, 128
    codes = torch.randint(-127, 128, (M, K), generator=g, device=gpu_dev, dtype=torch.int32).to(torch.int8)
    a = torch.randint(-100, 101, (L, R, K), generator=g, device=gpu_dev).to(BF16)
    rank_of = torch.randint(0, R, (L, N), generator=g, device=gpu_dev)
    b = torch.zeros(L, N, R, device=gpu_dev).scatter_(2, rank_of[:, :, None], 1.0).to(BF16)
    ids = torch.randint(-1, L, (M // 8,), generator=g, device=gpu_dev).repeat_interleave(8)
    w = icq.QuantizedWeight(torch.zeros(N, K // (1 if bits == 8 else 2), dtype=torch.int8 if bits == 8 else torch.uint8, device=gpu_dev), torch.ones(N, device=gpu_dev))
    act = icq.QuantizedActivations.from_codes(codes, torch.ones(M, device=gpu_dev))
    y = icq.quantized_linear(act, w, adapters=icq.LowRankAdapters(a, b), groups=icq.group_rows(ids, L), out_dtype=F32)
    x = codes.float()
    for n in range(-1, L):
        at = (ids == n).nonzero()[:, 0]
        want = torch.zeros(at.shape[0], N, device=gpu_dev) if n < 0 else (x[at].double() @ a[n, rank_of[n]].double().T.contiguous()).float()
        assert torch.equal(y[at], want)
