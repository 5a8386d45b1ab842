"""Rows ordered by group: the order of given ids, the router's choice, and the
weighted way back, each against its definition.

Bounds.  Numbers of groups, places and pairs are equal.  Weights: x - max is
rounded once, which moves exp by |x - max| 2^-24 of it; exp itself is within
2^-22; a sum of n terms in fp32 is within n 2^-24 (lanes' own, then six
additions: n <= 22 for up to 1024 experts, whose terms carry the exponentials'
error as well); the quotient adds 2^-24.  Together (2 |x - max| + 2 4 + 24) 2^-24
of the weight with the largest |x - max| of the row, or fp32's smallest normal
number.  The weighted sum: at most k + 1 roundings of partial sums, each 2^-24
of the sum of magnitudes, and half a step of the result's type.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
STEP = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
INF = float("inf")


def order_of(ids, groups):
    """(ids, offsets, order, position) from the definition, pair by pair."""
    flat = ids.reshape(-1).tolist()
    flat = [i if 0 <= i < groups else -1 for i in flat]
    order, offsets = [], [0]
    lists = [[] for _ in range(groups)]
    for p, i in enumerate(flat):
        if i >= 0:
            lists[i].append(p)
    for own in lists:
        order += own
        offsets.append(len(order))
    position = [-1] * len(flat)
    for at, p in enumerate(order):
        position[p] = at
    order += [-1] * (len(flat) - len(order))
    return [torch.tensor(v, dtype=torch.int32) for v in (flat, offsets, order, position)]


def same(g, ids, groups):
    want = order_of(ids, groups)
    assert (g.rows, g.groups) == (ids.shape[0], groups)
    for got, w, name in zip((g.ids, g.offsets, g.order, g.position), want, ("ids", "offsets", "order", "position")):
        assert got.dtype == torch.int32 and torch.equal(got.cpu().reshape(-1), w), name


@pytest.mark.parametrize("rows,per_row,groups", [(0, 1, 5), (1, 1, 1), (1, 4, 64), (15, 3, 7), (16, 1, 2), (17, 2, 63), (64, 1, 65),
                                                 (100, 64, 130), (257, 6, 60), (1000, 1, 1024), (4097, 2, 256), (5000, 8, 300),
                                                 (40000, 3, 1000)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_group_rows(gpu_dev, rows, per_row, groups, dtype):
    import int_crush_converter_amd as icq
    g = torch.Generator().manual_seed(rows + groups)
    ids = torch.randint(-1, groups, (rows, per_row), generator=g).to(dtype)
    same(icq.group_rows(ids.to(gpu_dev), groups), ids, groups)
    if per_row == 1:
        same(icq.group_rows(ids[:, 0].to(gpu_dev), groups), ids, groups)


def test_group_rows_of_odd_ids(gpu_dev):
    """One group has all, none has any, numbers that are no group's, a view with strides, host ids."""
    import int_crush_converter_amd as icq
    for ids in (torch.full((300, 2), 4), torch.full((300, 2), -1), torch.full((70, 1), 9),
                torch.tensor([[2 ** 40, -2 ** 40, 2 ** 32], [2 ** 32 + 1, 3, 0]]), torch.arange(90).reshape(30, 3) % 5):
        same(icq.group_rows(ids.to(gpu_dev), 9), ids, 9)
    ids = torch.arange(120).reshape(30, 4) % 7
    same(icq.group_rows(ids.to(gpu_dev)[:, ::2], 7), ids[:, ::2], 7)
    same(icq.group_rows(ids, 7), ids, 7)
    lowest = torch.tensor([[-2 ** 31, 2 ** 31 - 1, 0]], dtype=torch.int32)
    same(icq.group_rows(lowest.to(gpu_dev), 3), lowest, 3)


def choice_of(x, top):
    """Ids by repeated search of the largest left, NaN first, -inf never."""
    ids = []
    for row in x.double().tolist():
        rank = sorted((i for i, v in enumerate(row) if v != -INF), key=lambda i: (0, 0.0, i) if row[i] != row[i] else (1, -row[i], i))
        ids.append((rank + [-1] * top)[:top])
    return torch.tensor(ids, dtype=torch.int64).reshape(-1, top)


def check_route(x, top, renormalize, groups, weights):
    ids = choice_of(x.cpu(), top)
    same(groups, ids, x.shape[1])
    v = x.cpu().double()
    chosen = torch.where(ids < 0, -INF, v.gather(1, ids.clamp(min=0)))
    peak = torch.where(torch.isfinite(v), v, -1e300).amax(1, keepdim=True)          # (subtracted first: 3e38 has no room for a log)
    total = torch.exp((chosen if renormalize else v) - peak).sum(1, keepdim=True)
    odd = (torch.isnan(v) | (v == INF)).any(1, keepdim=True)
    want = torch.where(ids < 0, 0.0, torch.where(odd, float("nan"), torch.exp(chosen - peak) / total))
    spread = torch.where(torch.isfinite(v), (v - peak).abs(), 0.0).amax(1, keepdim=True).clamp(max=110)    # (beyond: exp is 0)
    room = want * (2 * spread + 32) * 2.0 ** -24 + 2.0 ** -126
    got = weights.cpu().double()
    assert weights.dtype == F32 and tuple(weights.shape) == tuple(ids.shape)
    known = ~torch.isnan(want)
    assert torch.equal(torch.isnan(got), ~known)
    assert ((got - want).abs()[known] <= room[known]).all()


@pytest.mark.parametrize("tokens,experts,top", [(0, 8, 2), (1, 1, 1), (1, 64, 4), (3, 60, 6), (16, 65, 8), (17, 128, 1), (40, 200, 64),
                                                (33, 256, 8), (300, 512, 3), (100, 1000, 10), (70, 1024, 2), (4100, 40, 2),
                                                (2000, 8, 8)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_route(gpu_dev, tokens, experts, top, dtype):
    import int_crush_converter_amd as icq
    g = torch.Generator().manual_seed(tokens + experts)
    x = (torch.randn(tokens, experts, generator=g) * 2).to(dtype).to(gpu_dev)      # 16 bits: many equal ones
    for renormalize in (True, False):
        check_route(x, top, renormalize, *icq.route_tokens(x, top, renormalize=renormalize))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("experts", [40, 130, 1024])
def test_route_of_masked_and_odd_rows(gpu_dev, dtype, experts):
    import int_crush_converter_amd as icq
    g = torch.Generator().manual_seed(experts)
    low = torch.finfo(dtype).min
    x = torch.randn(80, experts, generator=g).to(dtype)
    x[0] = -INF                                                    # nothing left
    x[1, 1:] = -INF                                                # one left, fewer than the choices
    x[2, : experts // 2] = -INF
    x[3] = low                                                     # the lowest value is a value
    x[4, ::2] = low
    x[5] = 0.0
    x[5, ::3] = -0.0                                               # the two zeros are equal
    x[6, 7] = INF
    x[7, 9] = float("nan")
    x[8, 9], x[8, 3], x[8, 4] = float("nan"), INF, -INF
    x[9] = torch.finfo(dtype).max
    x[10, 5] = torch.finfo(dtype).max
    x[11, :] = -INF
    x[11, -1] = low
    x[12] = torch.finfo(dtype).tiny / 2                            # subnormal, all equal
    x[12, 11] = torch.finfo(dtype).tiny
    x[20:60] = -INF                                                # padding
    x = x.to(gpu_dev)
    for renormalize in (True, False):
        check_route(x, 6, renormalize, *icq.route_tokens(x, 6, renormalize=renormalize))
    view = torch.zeros(80, experts + 3, dtype=dtype, device=gpu_dev)
    view[:, 2:-1] = x
    check_route(x, 6, True, *icq.route_tokens(view[:, 2:-1], 6))
    check_route(x, 6, True, *icq.route_tokens(x.T.contiguous().T, 6))


@pytest.mark.parametrize("tokens,top,cols", [(0, 2, 8), (1, 1, 1), (1, 4, 4096), (3, 2, 7), (37, 3, 2901), (20, 8, 2048), (9, 64, 2056),
                                             (300, 6, 520), (5, 5, 5000)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_combine(gpu_dev, tokens, top, cols, dtype):
    import int_crush_converter_amd as icq
    g = torch.Generator().manual_seed(tokens + cols)
    ids = torch.randint(-1, 9, (tokens, top), generator=g)
    groups = icq.group_rows(ids.to(gpu_dev), 9)
    y = torch.randn(tokens * top, cols, generator=g).to(dtype)
    w = torch.rand(tokens, top, generator=g)
    w[ids < 0] = float("nan")                                      # the weight of no expert is not looked at
    r = torch.randn(tokens, cols, generator=g).to(dtype)
    last = int(groups.offsets[-1])
    y[last:] = float("nan")                                        # nor are the rows behind the last group
    at = groups.position.cpu().long()
    for residual in (None, r):
        got = icq.combine_experts(y.to(gpu_dev), groups, w.to(gpu_dev), None if residual is None else residual.to(gpu_dev))
        terms = torch.where((at >= 0)[:, :, None], w.double()[:, :, None] * y.double()[at.clamp(min=0)], 0.0) if tokens else torch.zeros(0, top, cols)
        want, size = terms.sum(1), terms.abs().sum(1)
        if residual is not None:
            want, size = want + r.double(), size + r.double().abs()
        assert got.dtype == dtype and tuple(got.shape) == (tokens, cols)
        room = size * (top + 1) * 2.0 ** -24
        smallest = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps       # a subnormal's step
        assert ((got.cpu().double() - want).abs() <= room + (want.abs() + room) * STEP[dtype] + smallest).all()


def test_combine_strides_and_bad_rows(gpu_dev):
    """Rows at any pitch and alignment; a row with Inf or NaN reaches its own token only."""
    import int_crush_converter_amd as icq
    g = torch.Generator().manual_seed(3)
    ids = torch.tensor([[0, 1], [1, 0], [1, 2], [2, 0]])
    groups = icq.group_rows(ids.to(gpu_dev), 3)
    w = torch.rand(4, 2, generator=g).to(gpu_dev)
    for dtype in (F32, BF16, F16):
        y, r = torch.randn(8, 70, generator=g).to(dtype).to(gpu_dev), torch.randn(4, 70, generator=g).to(dtype).to(gpu_dev)
        want = icq.combine_experts(y, groups, w, r)
        for pad in (1, 2, 5):
            yv, rv = torch.zeros(8, 70 + pad + 3, dtype=dtype, device=gpu_dev)[:, pad: pad + 70], torch.zeros(4, 90, dtype=dtype, device=gpu_dev)[:, pad: pad + 70]
            yv.copy_(y)
            rv.copy_(r)
            assert torch.equal(icq.combine_experts(yv, groups, w, rv), want)
        assert torch.equal(icq.combine_experts(y.T.contiguous().T, groups, w, r), want)
        bad = y.clone()
        bad[int(groups.position[2, 1]), 5] = float("nan")
        bad[int(groups.position[2, 0]), 6] = INF
        got = icq.combine_experts(bad, groups, w, r)
        assert torch.isnan(got[2, 5]) and torch.isinf(got[2, 6])
        got[2, 5:7] = want[2, 5:7]
        assert torch.equal(got, want)


def test_as_many_pairs_as_there_may_be(gpu_dev):
    """1048560 pairs: units of thousands of rows, and rows whose offsets pass 32 bits."""
    import int_crush_converter_amd as icq
    n = 1048560
    g = torch.Generator(device=gpu_dev).manual_seed(1)
    x = torch.randn(n, 5, generator=g, device=gpu_dev)
    groups, w = icq.route_tokens(x, 1)
    ids = x.argmax(1)
    order = torch.argsort(ids, stable=True)
    assert torch.equal(groups.ids[:, 0].long(), ids) and torch.equal(groups.order.long(), order) and (w == 1).all()
    assert torch.equal(groups.offsets.long(), torch.searchsorted(ids[order], torch.arange(6, device=gpu_dev)))
    assert torch.equal(groups.position[order, 0].long(), torch.arange(n, device=gpu_dev))
    again = icq.group_rows(torch.arange(n, device=gpu_dev).reshape(-1, 60) % 1023, 1023)
    want = torch.argsort(torch.arange(n, device=gpu_dev) % 1023, stable=True)
    assert torch.equal(again.order.long(), want)
    cols = 2056                                                    # 2 pieces of a row, 2.2e9 elements
    y = torch.zeros(n, cols, dtype=torch.float16, device=gpu_dev)
    y[:, 7] = (order % 64).half()
    y[:, -1] = 3.0
    out = icq.combine_experts(y, groups, w)
    assert torch.equal(out[:, 7], (torch.arange(n, device=gpu_dev) % 64).half()) and (out[:, -1] == 3).all()
    assert not out[:, 8:-1].any()


def test_host_tensors(gpu_dev):
    """Host tensors are copied to the GPU and floating-point results back; the order stays there."""
    import int_crush_converter_amd as icq
    g = torch.Generator().manual_seed(8)
    x, y, r = torch.randn(9, 20, generator=g), torch.randn(27, 40, generator=g), torch.randn(9, 40, generator=g)
    groups, w = icq.route_tokens(x, 3)
    on, won = icq.route_tokens(x.to(gpu_dev), 3)
    assert not w.is_cuda and torch.equal(w, won.cpu()) and torch.equal(groups.order, on.order)
    out = icq.combine_experts(y, groups, w, r)
    assert not out.is_cuda and torch.equal(out, icq.combine_experts(y.to(gpu_dev), on, won, r.to(gpu_dev)).cpu())


def test_other_stream_and_graph(gpu_dev):
    """Calls follow the current stream; a captured router and its way back give the eager result on every replay."""
    import int_crush_converter_amd as icq
    g = torch.Generator().manual_seed(4)
    for tokens in (5, 700):
        x = torch.randn(tokens, 60, generator=g).to(gpu_dev)
        y = torch.randn(tokens * 4, 300, generator=g).to(BF16).to(gpu_dev)

        def chain():
            groups, w = icq.route_tokens(x, 4)
            again = icq.group_rows(groups.ids, 60)
            return groups.ids, groups.order, groups.offsets, groups.position, w, again.order, icq.combine_experts(y, groups, w)

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
            x.copy_(torch.randn(tokens, 60, generator=g))
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in held]
            assert all(torch.equal(a, b) for a, b in zip(got, chain())), k


def test_two_graphs_at_once(gpu_dev):
    """Two captured routers, replayed on two streams at once, have workspaces of their own."""
    import int_crush_converter_amd as icq
    g = torch.Generator().manual_seed(6)
    xs = [torch.randn(3000, 100, generator=g).to(gpu_dev) for _ in range(2)]
    want = [[t.clone() for t in (lambda r: (r[0].ids, r[0].order, r[0].offsets, r[0].position, r[1]))(icq.route_tokens(x, 5))] for x in xs]
    graphs, held, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r = icq.route_tokens(x, 5)
        graphs.append(graph)
        held.append((r[0].ids, r[0].order, r[0].offsets, r[0].position, r[1]))
    torch.cuda.synchronize()
    for k in range(3):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for h, w in zip(held, want) for a, b in zip(h, w)), k
