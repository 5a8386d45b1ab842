"""expert_linear against the definition in 64 bits.

Bounds.  The integer sums are exact, so an fp32 result has the roundings of
the sum's conversion, of sa * sw, of their product and of the bias addition:
4 2^-24 of (|y| + |bias|), doubled for the intermediate values: 2^-21.  A
16-bit result is the fp32 result rounded once, bit for bit.  Every form
gives the same bits as quantized_linear with the expert's own weight.
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


class Layer:
    def __init__(self, dev, E, N, K, bits, asym, seed, scale_dtype=F16, bias_dtype=F32):
        import int_crush_converter_amd as icq
        g = torch.Generator().manual_seed(seed)
        lo, hi = (-8, 8) if bits == 4 else (-128, 128)
        self.g, self.dev, self.E, self.N, self.K = g, dev, E, N, K
        self.q = torch.randint(lo, hi, (E, N, K), generator=g).to(torch.int8)
        self.z = torch.randint(lo, hi, (E, N), generator=g).to(torch.int8) if asym else None
        self.s = (torch.rand(E, N, generator=g) * 0.01 + 1e-4).to(scale_dtype)
        self.bias = torch.randn(E, N, generator=g).to(bias_dtype)
        self.each = [icq.QuantizedWeight((pack4(self.q[e]) if bits == 4 else self.q[e]).to(dev), self.s[e].to(dev),
                                         None if self.z is None else self.z[e].to(dev), in_features=K) for e in range(E)]
        self.w = icq.ExpertWeight(self.each)

    def rows(self, n):
        a = torch.randint(-128, 128, (n, self.K), generator=self.g).to(torch.int8)
        return a, torch.rand(n, generator=self.g) * 0.01 + 1e-4

    def want(self, a, sa, ids, gather, bias):
        """[rows * top, N] in the order of the groups, fp64."""
        E, top = self.E, ids.shape[1]
        flat = torch.where((ids < 0) | (ids >= E), E, ids).reshape(-1)
        order = torch.argsort(flat, stable=True)
        order = order[: int((flat < E).sum())]
        y = torch.empty(order.shape[0], self.N, dtype=torch.float64)
        for e in range(E):
            at = (flat[order] == e).nonzero()[:, 0]
            if at.shape[0]:
                src = order[at] // top if gather else at
                w = self.q[e].double() - (0 if self.z is None else self.z[e].double()[:, None])
                y[at] = (a[src].double() @ w.T) * sa[src].double()[:, None] * self.s[e].double()
                if bias:
                    y[at] += self.bias[e].double()
        return y, order


def skewed(g, rows, top, E):
    """Ids with a few popular experts, one without rows, some pairs of none."""
    p = 1.0 / (1 + torch.arange(E).double())
    if E > 2:
        p[1] = 0
    ids = torch.multinomial(p, rows * top, replacement=True, generator=g).reshape(rows, top)
    ids[torch.rand(rows, top, generator=g) < 0.1] = -1
    return ids


SIZES = [  # rows, top, E, N, K
    (1, 1, 1, 1, 1), (1, 2, 4, 16, 128), (3, 2, 5, 17, 127), (1, 8, 64, 48, 300), (40, 3, 6, 100, 65), (64, 2, 4, 40, 200),
    (33, 4, 3, 129, 384), (20, 2, 1000, 33, 129), (150, 2, 2, 64, 1000), (300, 1, 2, 130, 257), (500, 2, 3, 264, 640), (700, 2, 4, 300, 130),
    (900, 2, 3, 512, 100), (1200, 2, 2, 260, 1153), (2100, 1, 1, 1000, 64), (513, 3, 70, 96, 520), (1500, 2, 300, 24, 72),
    (1000, 2, 300, 40, 200), (9000, 4, 256, 130, 65), (70000, 4, 300, 17, 40), (1600, 1, 2, 33000, 128), (300, 2, 260, 72, 640),
    (100, 2, 8, 3000, 130), (900, 1, 6, 2000, 260), (2000, 4, 40, 700, 128), (560, 2, 20, 1500, 200), (70000, 2, 100, 700, 72), (20, 1, 54, 3900, 120),
    (260, 1, 300, 200, 1100), (9000, 4, 64, 260, 520), (4600, 4, 16, 1100, 1153),
]


@pytest.mark.parametrize("rows,top,E,N,K", SIZES)
@pytest.mark.parametrize("bits,asym", [(4, True), (4, False), (8, True), (8, False)])
def test_against_64_bits(gpu_dev, rows, top, E, N, K, bits, asym):
    import int_crush_converter_amd as icq
    layer = Layer(gpu_dev, E, N, K, bits, asym, rows + N + K)
    ids = skewed(layer.g, rows, top, E)
    groups = icq.group_rows(ids.to(gpu_dev), E)
    for gather in (True, False):
        a, sa = layer.rows(rows if gather else rows * top)
        act = icq.QuantizedActivations.from_codes(a.to(gpu_dev), sa.to(gpu_dev))
        want, order = layer.want(a, sa, ids, gather, gather)
        y = icq.expert_linear(act, layer.w, groups, layer.bias.to(gpu_dev) if gather else None, gather=gather, out_dtype=F32)
        assert y.dtype == F32 and tuple(y.shape) == (rows * top, N)
        room = want.abs() + (layer.bias.double().abs()[ids.reshape(-1)[order]] if gather else 0)
        assert ((y[: order.shape[0]].cpu().double() - want).abs() <= TOL * room + 1e-12).all()


def test_sizes_reach_every_form(gpu_dev):
    import int_crush_converter_amd._native as nat
    form = lambda bits: {nat.lib().ic_expert_form(bits, r * t, e, n, k) for r, t, e, n, k in SIZES}      # noqa: E731
    assert form(4) == {1, 2, 32, 64, 256} and form(8) == {1, 2, 128, 256}


@pytest.mark.parametrize("rows,top,E,N,K", [(3, 2, 5, 40, 200), (90, 2, 4, 37, 130), (700, 2, 4, 260, 520), (1500, 2, 2, 264, 300), (1500, 2, 2, 261, 300),
                                            (4600, 2, 16, 1700, 300)])
def test_output_types_and_the_experts_own_products(gpu_dev, rows, top, E, N, K):
    """16-bit results are the fp32 ones rounded once; each row has the bits of quantized_linear with its expert's weight."""
    import int_crush_converter_amd as icq
    for bits, asym, bdt, sdt in ((4, True, F32, F32), (8, False, BF16, F16), (8, True, F16, F16), (4, False, F32, F16)):
        layer = Layer(gpu_dev, E, N, K, bits, asym, rows + N, sdt, bdt)
        ids = skewed(layer.g, rows, top, E)
        groups = icq.group_rows(ids.to(gpu_dev), E)
        a, sa = layer.rows(rows)
        act = icq.QuantizedActivations.from_codes(a.to(gpu_dev), sa.to(gpu_dev))
        bias = layer.bias.to(gpu_dev)
        y = icq.expert_linear(act, layer.w, groups, bias, gather=True, out_dtype=F32)
        edges = groups.offsets.tolist()
        y = y[: edges[-1]]
        for dtype in (BF16, F16):
            got = icq.expert_linear(act, layer.w, groups, bias, gather=True, out_dtype=dtype)
            assert got.dtype == dtype and torch.equal(got[: edges[-1]], y.to(dtype))
        for e in range(E):
            src = groups.order[edges[e]: edges[e + 1]].long() // top
            if src.numel():
                own = icq.QuantizedActivations.from_codes(a.to(gpu_dev)[src], sa.to(gpu_dev)[src])
                assert torch.equal(icq.quantized_linear(own, layer.each[e], bias[e], out_dtype=F32), y[edges[e]: edges[e + 1]])


@pytest.mark.parametrize("rows,E", [(20, 4), (300, 4), (900, 3), (2400, 2)])
def test_rows_behind_the_last_and_out(gpu_dev, rows, E):
    """`out` of any pitch and alignment gets the same bits; pairs of no expert, and what lies beside, are left as they were."""
    import int_crush_converter_amd as icq
    layer = Layer(gpu_dev, E, 72, 200, 4, True, rows)
    ids = skewed(layer.g, rows, 2, E)
    ids[rows // 2:] = -1
    groups = icq.group_rows(ids.to(gpu_dev), E)
    a, sa = layer.rows(rows * 2)
    sa[int(groups.offsets[-1]):] = float("nan")
    act = icq.QuantizedActivations.from_codes(a.to(gpu_dev), sa.to(gpu_dev))
    last = int(groups.offsets[-1])
    y = icq.expert_linear(act, layer.w, groups, gather=False, out_dtype=BF16)
    for pad, at in ((0, 0), (8, 8), (5, 3), (24, 16)):
        hold = torch.full((rows * 2, 72 + pad + at), 7.0, dtype=BF16, device=gpu_dev)
        out = hold[:, at: at + 72]
        assert icq.expert_linear(act, layer.w, groups, gather=False, out=out) is out
        assert torch.equal(out[:last], y[:last])
        hold[:last, at: at + 72] = 7.0
        assert (hold == 7.0).all()
    none = icq.group_rows(torch.full((rows, 2), -1, device=gpu_dev), E)
    hold = torch.full((rows * 2, 72), 7.0, device=gpu_dev)
    icq.expert_linear(act, layer.w, none, gather=False, out=hold)
    assert (hold == 7.0).all()
    none = icq.group_rows(torch.zeros(0, 2, dtype=torch.int32, device=gpu_dev), E)
    act = icq.QuantizedActivations.from_codes(a[:0].to(gpu_dev), sa[:0].to(gpu_dev))
    for gather in (True, False):
        assert tuple(icq.expert_linear(act, layer.w, none, gather=gather).shape) == (0, 72)


@pytest.mark.parametrize("rows,E", [(10, 3), (400, 2), (1300, 2)])
def test_bad_rows_stay_alone(gpu_dev, rows, E):
    """A row whose scale is NaN gives NaN in its own places only."""
    import int_crush_converter_amd as icq
    layer = Layer(gpu_dev, E, 40, 130, 8, True, rows)
    ids = torch.randint(0, E, (rows, 2), generator=layer.g)
    groups = icq.group_rows(ids.to(gpu_dev), E)
    a, sa = layer.rows(rows)
    run = lambda s: icq.expert_linear(icq.QuantizedActivations.from_codes(a.to(gpu_dev), s.to(gpu_dev)), layer.w, groups,     # noqa: E731
                                      gather=True, out_dtype=F32)
    y = run(sa)
    bad = sa.clone()
    bad[rows // 2] = float("nan")
    got = run(bad)
    mine = groups.position[rows // 2].long()
    assert torch.isnan(got[mine]).all()
    got[mine] = y[mine]
    assert torch.equal(got, y)


@pytest.mark.parametrize("bits", [4, 8])
def test_extremes_of_the_sums(gpu_dev, bits):
    """K = 65536 with the largest codes of one sign: |sum| up to 2^31 - and the zero-point's share."""
    import int_crush_converter_amd as icq
    K, N, E = 65536, 20, 2
    lo, hi = (-8, 7) if bits == 4 else (-128, 127)
    q = torch.stack((torch.full((N, K), lo), torch.full((N, K), hi))).to(torch.int8)
    z = torch.stack((torch.full((N,), hi), torch.full((N,), lo))).to(torch.int8)
    s = torch.full((E, N), 0.5, dtype=F32)
    w = icq.ExpertWeight([icq.QuantizedWeight((pack4(q[e]) if bits == 4 else q[e]).to(gpu_dev), s[e].to(gpu_dev), z[e].to(gpu_dev)) for e in range(E)])
    for rows in (4, 600):
        a = torch.full((rows, K), -128, dtype=torch.int8)
        a[1::2] = 127
        ids = (torch.arange(rows) // 2 % 2).reshape(-1, 1)
        groups = icq.group_rows(ids.to(gpu_dev), E)
        act = icq.QuantizedActivations.from_codes(a.to(gpu_dev), torch.ones(rows, device=gpu_dev))
        y = icq.expert_linear(act, w, groups, gather=True, out_dtype=F32).cpu().double()
        src = groups.order.cpu().long()
        e = ids.reshape(-1)[src]
        want = a[src, 0].double() * K * (q[e, 0, 0].double() - z[e, 0].double()) * 0.5
        assert ((y - want[:, None]).abs() <= TOL * want.abs()[:, None]).all()


def test_gathered_rows_past_two_gigabytes(gpu_dev):
    """Offsets of gathered rows that pass 31 bits, in a form of each kind; at 2^32 bytes the call is refused."""
    import int_crush_converter_amd as icq
    K, N = 65536, 16
    rows = 40000                                                   # 2.6 GB of codes
    data = torch.zeros(rows, K, dtype=torch.int8, device=gpu_dev)
    meta = torch.zeros(2, rows, device=gpu_dev)
    act = icq.QuantizedActivations(data, meta, K, (rows,))
    act.scales.fill_(1.0)
    data[:, 5] = (torch.arange(rows, device=gpu_dev) % 101 - 50).to(torch.int8)
    q = torch.zeros(N, K, dtype=torch.int8)
    q[:, 5] = torch.arange(N)
    for bits in (4, 8):
        q4 = q.clamp(max=7)
        w = icq.ExpertWeight([icq.QuantizedWeight((pack4(q4) if bits == 4 else q).to(gpu_dev), torch.ones(N, device=gpu_dev))] * 2)
        want = (data[:, 5].double()[:, None] * (q4 if bits == 4 else q)[:, 5].double().to(gpu_dev))
        for some in (None, 30):
            ids = torch.full((rows, 1), -1, device=gpu_dev)
            if some is None:
                ids[:] = torch.arange(rows, device=gpu_dev)[:, None] % 2
            else:
                ids[-some:] = 1
            groups = icq.group_rows(ids, 2)
            last = int(groups.offsets[-1])
            y = icq.expert_linear(act, w, groups, gather=True, out_dtype=F32)[:last]
            assert torch.equal(y.double(), want[groups.order[:last].long()])
    del data, act
    rows = 65536
    act = icq.QuantizedActivations(torch.empty(rows, K, dtype=torch.int8, device=gpu_dev), torch.empty(2, rows, device=gpu_dev), K, (rows,))
    groups = icq.group_rows(torch.zeros(rows, 1, dtype=torch.int32, device=gpu_dev), 2)
    with pytest.raises(RuntimeError, match="2\\^32"):
        icq.expert_linear(act, w, groups, gather=True)


def test_permuted_layers_and_copies(gpu_dev):
    """Experts that the converter permuted; the weight is a copy."""
    import int_crush_converter_amd as icq
    g = torch.Generator().manual_seed(9)
    E, N, K = 3, 24, 130
    q = torch.randint(-8, 8, (E, N, K), generator=g).to(torch.int8)
    perm = [torch.randperm(128, generator=g) for _ in range(E)]
    s = torch.full((N,), 0.01, device=gpu_dev)
    stored = [torch.cat((q[e][:, perm[e]], q[e][:, 128:]), 1) for e in range(E)]
    plain = [icq.QuantizedWeight(pack4(q[e]).to(gpu_dev), s) for e in range(E)]
    permuted = [icq.QuantizedWeight(pack4(stored[e]).to(gpu_dev), s, permutation=perm[e].to(gpu_dev)) for e in range(E)]
    act = icq.quantize_activations(torch.randn(50, K, generator=g).to(gpu_dev))
    groups = icq.group_rows(torch.randint(0, E, (50,), generator=g).to(gpu_dev), E)
    a, b = icq.ExpertWeight(plain), icq.ExpertWeight(permuted)
    for w in plain:
        w.tiles.zero_()
    assert torch.equal(icq.expert_linear(act, a, groups, gather=True), icq.expert_linear(act, b, groups, gather=True))


def test_feed_forward_of_experts(gpu_dev):
    """The operators as they are used, against 64 bits: router, up projections of gathered tokens, down projections of
    ordered rows, the way back; on another stream and from a graph.

    The down projections' inputs are taken as the package quantised them, so what is compared is each product: bounds as
    above, with the weights' (32 + 2 max|x|) 2^-24 and the two roundings to bfloat16 (2^-8 of each term of the sum, and of it)."""
    import int_crush_converter_amd as icq
    for T in (3, 60, 700):
        g = torch.Generator().manual_seed(T)
        up = Layer(gpu_dev, 8, 96, 128, 4, True, T + 1)
        down = Layer(gpu_dev, 8, 128, 96, 8, True, T + 2)
        x = torch.randn(T, 128, generator=g).to(BF16).to(gpu_dev)
        logits = torch.randn(T, 8, generator=g).to(gpu_dev)
        logits[:: 3] = -float("inf")
        kept = {}

        def layer():
            groups, w = icq.route_tokens(logits, 2)
            act = icq.quantize_activations(x)
            inner = icq.expert_linear(act, up.w, groups, gather=True)
            act2 = icq.quantize_activations(torch.nn.functional.silu(inner))
            z = icq.expert_linear(act2, down.w, groups, gather=False)
            kept.update(groups=groups, w=w, act=act, inner=inner, act2=act2, z=z)
            return icq.combine_experts(z, groups, w, x)

        y = layer()
        groups, last = kept["groups"], int(kept["groups"].offsets[-1])
        ids = groups.ids.cpu().long()
        want, _ = up.want(kept["act"].codes.cpu(), kept["act"].scales.cpu(), ids, True, False)
        err = (kept["inner"][:last].cpu().double() - want).abs()
        assert (err <= want.abs() * (2.0 ** -8 + 2 * TOL) + 1e-12).all()
        want, order = down.want(kept["act2"].codes.cpu(), kept["act2"].scales.cpu(), ids, False, False)
        p = torch.where(ids < 0, 0.0, torch.softmax(torch.where(ids < 0, -float("inf"), logits.cpu().double().gather(1, ids.clamp(min=0))), 1).nan_to_num())
        total, size = x.cpu().double(), x.cpu().double().abs()
        for at, pair in enumerate(order.tolist()):
            t, j = divmod(pair, 2)
            total[t] += p[t, j] * want[at]
            size[t] += (p[t, j] * want[at]).abs()
        assert ((y.cpu().double() - total).abs() <= size * (2.0 ** -8 + 2.0 ** -17) + total.abs() * 2.0 ** -8).all()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = layer()
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(other, y)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = layer()
        for k in range(4):
            logits.copy_(torch.randn(T, 8, generator=g))
            x.copy_(torch.randn(T, 128, generator=g).to(BF16))
            graph.replay()
            torch.cuda.synchronize()
            got = held.clone()
            assert torch.equal(got, layer()), k
