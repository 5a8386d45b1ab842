"""Refusals of the operators on grouped rows and adapters: no GPU.  Tensors
are stand-ins where a check comes after they would be on one."""

from __future__ import annotations

import ctypes
import os

import pytest
import torch

import int_crush_converter_amd as icq
from int_crush_converter_amd import _native as nat
from int_crush_converter_amd import activations, adapters, experts, groups, linear

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(nat.LIB_PATH):
        from int_crush_converter_amd import build
        build.build()
    nat.load(require_gpu=False)
    return nat._lib


@pytest.fixture
def calls(monkeypatch):
    """The package with its calls recorded and every tensor taken as the current GPU's."""
    made = []
    for mod in (activations, adapters, experts, groups, linear):
        monkeypatch.setattr(mod, "call", lambda name, *args: made.append(name))
    monkeypatch.setattr(nat, "on_gpu", lambda name, t: t)
    monkeypatch.setattr(nat, "to_gpu", lambda t: t)
    monkeypatch.setattr(nat, "stream_for", lambda *t: 0)
    return made


def rows_of(rows, per_row, n):
    return groups.RowGroups._empty(rows, per_row, n, torch.device("cpu"))


def act(rows, K):
    return icq.QuantizedActivations(torch.zeros(rows, -(-K // 128) * 128, dtype=torch.int8), torch.zeros(2, rows), K, (rows,))


def weight(N, K, bits=8, zeros=False, kind=0):
    w = icq.QuantizedWeight.__new__(icq.QuantizedWeight)
    w.tiles = torch.zeros(-(-N // 16) * -(-K // 128) * (2048 if bits == 8 else 1024), dtype=torch.uint8)
    w.scales, w.scale_kind = torch.ones(N, dtype=torch.float16 if kind == 0 else F32), kind
    w.zero_points = torch.zeros(N, dtype=torch.int8) if zeros else None
    w.bits, w.in_features, w.out_features = bits, K, N
    return w


def test_rows_of_groups_are_made_by_calls():
    with pytest.raises(TypeError, match="group_rows"):
        icq.RowGroups()


def test_refused_ids(calls):
    for ids in (torch.zeros(3), torch.zeros(2, 2, 2, dtype=torch.int32), torch.tensor(3), torch.zeros(3, dtype=torch.int16)):
        with pytest.raises(ValueError, match="int32 or int64"):
            icq.group_rows(ids, 4)
    for shape, n in (((3,), 0), ((3,), 1025), ((3, 65), 4), ((3, 0), 4), ((1048561,), 4), ((20000, 60), 4)):
        with pytest.raises(ValueError, match="at most"):
            icq.group_rows(torch.zeros(shape, dtype=torch.int32), n)
    assert not calls
    icq.group_rows(torch.zeros(1048560, dtype=torch.int32), 1024)
    assert calls == ["ic_group_rows"]


def test_refused_logits(calls):
    with pytest.raises(ValueError, match="tokens, experts"):
        icq.route_tokens(torch.zeros(8), 2)
    for top in (0, 9, -1):
        with pytest.raises(ValueError, match="top"):
            icq.route_tokens(torch.zeros(4, 8), top)
    with pytest.raises(TypeError):
        icq.route_tokens(torch.zeros(4, 8, dtype=torch.float64), 2)
    for shape, top in (((2, 1025), 2), ((2, 100), 65), ((300000, 8), 4)):
        with pytest.raises(ValueError, match="at most"):
            icq.route_tokens(torch.zeros(shape, dtype=BF16), top)
    assert not calls


def test_refused_sums(calls):
    g = rows_of(5, 2, 4)
    y, w = torch.zeros(10, 24, dtype=BF16), torch.zeros(5, 2)
    icq.combine_experts(y, g, w, torch.zeros(5, 24, dtype=BF16))
    assert calls == ["ic_combine_rows"]
    for bad in (torch.zeros(9, 24), torch.zeros(10, 0), torch.zeros(10, 2, 24)):
        with pytest.raises(ValueError, match="expected y"):
            icq.combine_experts(bad, g, w)
    for bad in (torch.zeros(5, 3), torch.zeros(10), torch.zeros(5, 2, dtype=torch.int32)):
        with pytest.raises(ValueError, match="weights"):
            icq.combine_experts(y, g, bad)
    for bad in (torch.zeros(5, 24), torch.zeros(10, 24, dtype=BF16), torch.zeros(5, 23, dtype=BF16)):
        with pytest.raises(ValueError, match="residual"):
            icq.combine_experts(y, g, w, bad)
    with pytest.raises(TypeError):
        icq.combine_experts(y.double(), g, w)
    assert len(calls) == 1


def test_refused_experts(calls):
    for layers in ([], [weight(16, 64)] * 1025):
        with pytest.raises(ValueError, match="experts"):
            icq.ExpertWeight(layers)
    for other in (weight(16, 65), weight(17, 64), weight(16, 64, bits=4), weight(16, 64, zeros=True), weight(16, 64, kind=1)):
        with pytest.raises(ValueError, match="expert 1 differs"):
            icq.ExpertWeight([weight(16, 64), other])
    w, g = icq.ExpertWeight([weight(16, 64)] * 4), rows_of(5, 2, 4)
    icq.expert_linear(act(5, 64), w, g, gather=True)
    icq.expert_linear(act(10, 64), w, g, torch.zeros(4, 16), gather=False)
    assert calls == ["ic_expert_linear"] * 2
    for x, gather in ((act(10, 64), True), (act(5, 64), False), (act(0, 64), True)):
        with pytest.raises(ValueError, match="rows of activations"):
            icq.expert_linear(x, w, g, gather=gather)
    with pytest.raises(ValueError, match="features"):
        icq.expert_linear(act(5, 65), w, g, gather=True)
    with pytest.raises(ValueError, match="grouped among"):
        icq.expert_linear(act(5, 64), w, rows_of(5, 2, 5), gather=True)
    for bias in (torch.zeros(16), torch.zeros(4, 15), torch.zeros(16, 4)):
        with pytest.raises(ValueError, match="bias"):
            icq.expert_linear(act(5, 64), w, g, bias, gather=True)
    with pytest.raises(TypeError):
        icq.expert_linear(act(5, 64), w, g, gather=True, out_dtype=torch.float64)
    for out in (torch.zeros(5, 16), torch.zeros(10, 17), torch.zeros(16, 10).T, torch.zeros(1, 16).expand(10, 16)):
        with pytest.raises(ValueError, match="out must be"):
            icq.expert_linear(act(5, 64), w, g, gather=True, out=out)
    with pytest.raises(TypeError):
        icq.expert_linear(act(5, 64), w, g, gather=True, out=torch.zeros(10, 16, dtype=torch.float64))
    assert len(calls) == 2


def adapter(n, r, N, K):
    a = icq.LowRankAdapters.__new__(icq.LowRankAdapters)
    a.down = a.up = torch.zeros(16, dtype=torch.uint8)
    a.scaling, a.code, a.count, a.rank, a.in_features, a.out_features = torch.ones(n), 1, n, r, K, N
    return a


def test_refused_adapters(calls):
    ok_a, ok_b = torch.zeros(2, 4, 64, dtype=BF16), torch.zeros(2, 16, 4, dtype=BF16)
    for a, b in ((ok_a[0], ok_b), (ok_a, ok_b[0]), (ok_a, torch.zeros(3, 16, 4, dtype=BF16)), (ok_a, torch.zeros(2, 16, 5, dtype=BF16))):
        with pytest.raises(ValueError, match="expected a"):
            icq.LowRankAdapters(a, b)
    for a, b in ((ok_a.float(), ok_b.float()), (ok_a, ok_b.half())):
        with pytest.raises(TypeError):
            icq.LowRankAdapters(a, b)
    for n, r, N, K in ((0, 4, 16, 64), (2, 0, 16, 64), (2, 129, 16, 64), (2, 4, 16, 0), (2, 4, 16, 65537), (2, 4, 0, 64), (1025, 1, 1, 1)):
        with pytest.raises(ValueError, match="adapters of rank"):
            icq.LowRankAdapters(torch.zeros(n, r, K, dtype=BF16), torch.zeros(n, N, r, dtype=BF16))
    for value in (float("nan"), float("inf")):
        odd = ok_b.clone()
        odd[1, 3, 2] = value
        with pytest.raises(ValueError, match="Inf or NaN"):
            icq.LowRankAdapters(ok_a, odd)
    with pytest.raises(ValueError, match="scalings"):
        icq.LowRankAdapters(ok_a, ok_b, torch.ones(3))
    w, ad = weight(16, 64), adapter(2, 4, 16, 64)
    icq.quantized_linear(act(5, 64), w, adapters=ad, groups=rows_of(5, 1, 2))
    assert calls == ["ic_adapted_linear"]
    for bad in (adapter(2, 4, 17, 64), adapter(2, 4, 16, 63)):
        with pytest.raises(ValueError, match="adapters are"):
            icq.quantized_linear(act(5, 64), w, adapters=bad, groups=rows_of(5, 1, 2))
    for g in (rows_of(4, 1, 2), rows_of(5, 2, 2), rows_of(5, 1, 3)):
        with pytest.raises(ValueError, match="groups are of"):
            icq.quantized_linear(act(5, 64), w, adapters=ad, groups=g)
    with pytest.raises(ValueError, match="group_rows"):
        icq.quantized_linear(act(5, 64), w, adapters=ad)
    with pytest.raises(ValueError, match="expert_linear"):
        icq.quantized_linear(act(5, 64), w, groups=rows_of(5, 1, 2))
    assert len(calls) == 1


def test_operands_elsewhere(monkeypatch):
    """Every operand is asked where it lies; host tensors stand for another device."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    g, w = rows_of(5, 2, 4), None
    with pytest.raises(ValueError, match="current device"):
        icq.ExpertWeight([weight(16, 64)])
    monkeypatch.setattr(nat, "stream_for", lambda *t: 0)
    w = icq.ExpertWeight([weight(16, 64)] * 4)
    monkeypatch.undo()
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(nat, "to_gpu", lambda t: t)
    for f in (lambda: icq.expert_linear(act(5, 64), w, g, gather=True),
              lambda: icq.group_rows(torch.zeros(3, dtype=torch.int32), 4),
              lambda: icq.route_tokens(torch.zeros(3, 8), 2),
              lambda: icq.combine_experts(torch.zeros(10, 8), g, torch.zeros(5, 2)),
              lambda: icq.quantized_linear(act(5, 64), weight(16, 64), adapters=adapter(2, 4, 16, 64), groups=rows_of(5, 1, 2))):
        with pytest.raises(ValueError, match="current device is cuda:0"):
            f()


def test_sizes_of_the_library(L):
    assert L.ic_group_workspace_bytes(0, 5) == 0 and L.ic_group_workspace_bytes(1, 5) == 16
    assert L.ic_group_workspace_bytes(17, 64) == 2 * 64 * 2 and L.ic_group_workspace_bytes(1048560, 1024) <= 256 * 1024 * 2
    assert L.ic_group_workspace_bytes(10, 1025) == 0
    for rows in (1, 16, 17, 4000, 4096, 4097, 8191, 100000, 1048560):
        assert L.ic_group_workspace_bytes(rows, 7) <= 4 * groups.RowGroups._empty(rows, 1, 7, torch.device("cpu")).scratch
    assert L.ic_adapter_down_bytes(3, 12, 130) == 3 * 16 * 256 * 2 and L.ic_adapter_up_bytes(3, 17, 33, 1) == 3 * 2 * 2 * 1024
    assert L.ic_adapter_up_bytes(3, 17, 33, 2) == 3 * 2 * 2 * 3072 and L.ic_adapter_up_bytes(3, 17, 33, 0) == 0
    assert L.ic_adapted_linear_workspace_bytes(7, 12) == 8 * 128
    assert L.ic_adapter_up_bytes(1024, 1048560, 128, 1) == 1024 * 1048560 * 128 * 2           # past 32 bits


def test_refusals_of_the_library(L):
    one = ctypes.c_void_p(16)          # an address that no refused call touches
    route = lambda **k: L.ic_route_tokens(one, k.get("dtype", 0), k.get("tokens", 4), k.get("experts", 8), k.get("ld", 8),      # noqa: E731
                                          k.get("top", 2), 1, one, one, k.get("offsets", one), one, one, one, None)
    assert route(dtype=3) == -1 and route(top=0) == -1 and route(top=9) == -1 and route(ld=7) == -1 and route(experts=0) == -1
    assert route(tokens=-1) == -1 and route(offsets=None) == -1 and route(experts=1025, ld=1025) == -3
    assert route(tokens=1048560) == -3 and route(tokens=1 << 40, top=1) == -3 and route(experts=100, ld=100, top=65) == -3
    rows = lambda **k: L.ic_group_rows(k.get("ids", one), 0, k.get("rows", 4), k.get("per", 2), k.get("groups", 8), one, one, one, one,     # noqa: E731
                                       k.get("ws", one), None)
    assert rows(ids=None) == -1 and rows(ws=None) == -1 and rows(per=0) == -1 and rows(groups=0) == -1 and rows(groups=2000) == -3
    assert rows(ws=ctypes.c_void_p(8)) == -1
    assert rows(rows=1 << 62, per=64) == -3
    comb = lambda **k: L.ic_combine_rows(k.get("y", one), k.get("dtype", 1), k.get("tokens", 4), k.get("top", 2), k.get("cols", 64),         # noqa: E731
                                         k.get("ldy", 64), one, one, k.get("res"), k.get("ldr", 0), one, k.get("ldo", 64), None)
    assert comb(y=None) == -1 and comb(dtype=4) == -1 and comb(cols=0) == -1 and comb(ldy=63) == -1 and comb(ldo=63) == -1
    assert comb(res=one, ldr=63) == -1 and comb(top=65) == -3 and comb(tokens=1048560) == -3 and comb(tokens=0) == 0
    assert comb(tokens=1 << 40, top=1) == -3 and comb(cols=1 << 21, ldy=1 << 21, ldo=1 << 21) == -3
    ex = lambda **k: L.ic_expert_linear(one, k.get("lda", 128), one, None, k.get("arows", 4), k.get("offsets", one), k.get("order", one),     # noqa: E731
                                        k.get("top", 2), k.get("groups", 3), k.get("rows", 8), one, k.get("bits", 4), one, 0, k.get("zp"),
                                        None, 0, k.get("N", 8), k.get("K", 64), one, k.get("out", 1), k.get("ldo", 8), None)
    assert ex(bits=3) == -1 and ex(out=5) == -1 and ex(lda=64) == -1 and ex(ldo=7) == -1 and ex(zp=one) == -1 and ex(offsets=None) == -1
    assert ex(order=None) == -1 and ex(top=0) == -1 and b"differ" in L.ic_last_error()
    assert ex(groups=0) == -1 and ex(groups=1025) == -1 and ex(top=-1) == -1 and ex(arows=0) == -1
    assert ex(K=65537, lda=65664) == -3 and ex(rows=1048561) == -3 and ex(rows=0) == 0
    assert ex(arows=1 << 19, lda=1 << 13) == -3 and b"2^32" in L.ic_last_error()
    ad = lambda **k: L.ic_adapted_linear(one, 128, one, None, k.get("M", 4), one, 4, one, 0, None, None, 0, 8, 64, k.get("down", one), one,    # noqa: E731
                                         k.get("dtype", 1), k.get("n", 3), k.get("rank", 8), one, k.get("ids", one), one, one,
                                         k.get("ws", one), one, 1, k.get("ldo", 8), None)
    assert ad(down=None) == -1 and ad(dtype=0) == -1 and ad(n=0) == -1 and ad(n=1025) == -1 and ad(rank=0) == -1 and ad(rank=129) == -1
    assert ad(ids=None) == -1 and ad(ws=None) == -1 and ad(ws=ctypes.c_void_p(8)) == -1 and ad(ldo=7) == -1 and ad(M=0) == 0
    pack = lambda **k: L.ic_adapter_pack(k.get("a", one), one, k.get("dtype", 1), k.get("n", 2), k.get("rank", 4), k.get("N", 8), k.get("K", 8), one,             # noqa: E731
                                         k.get("up", one), None)
    assert pack(a=None) == -1 and pack(n=0) == -1 and pack(K=0) == -1 and pack(up=ctypes.c_void_p(8)) == -1
    assert pack(dtype=0) == -1 and pack(n=1024, N=1048560) == -3
    assert pack(n=1025) == -3 and pack(rank=129) == -3 and pack(K=65537) == -3
    form = L.ic_expert_form
    assert form(4, -1, 4, 8, 8) == -1 and form(4, 4, 0, 8, 8) == -1 and form(3, 4, 4, 8, 8) == -1 and form(4, 4, 4, 8, 0) == -1
