"""The operators that run quantised experts and adapters, as cases that can be timed and compared.

Four operators, each in a plain form (elementary torch operations in 32 bits)
and as the package's own calls: the router, which chooses experts for each
token and orders the chosen (token, expert) pairs by expert; the products of
such ordered rows of 8-bit activations with the INT4 / INT8 weights of their
experts; the weighted sum that brings the experts' rows back to their tokens;
and the product with one shared quantised weight beside which each row adds
the low-rank adapter of its own request.  ``exact`` restates each in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # one token's router: launches and latency count
        {"name": "route_1x64_top4", "kind": "route", "rows": 1, "experts": 64, "top": 4, "renormalize": True,
         "padded": 0.0, "dtype": "bfloat16"},
        # a long batch of prompts, a tenth of whose rows are padding (no expert admitted)
        {"name": "route_8191x256_top8", "kind": "route", "rows": 8191, "experts": 256, "top": 8, "renormalize": False,
         "padded": 0.1, "dtype": "float32"},
        # a few tokens of odd width back in the residual stream
        {"name": "combine_37x2901_top3", "kind": "combine", "rows": 37, "experts": 10, "top": 3, "out": 2901,
         "residual": False, "dtype": "float16"},
        # a long prompt back in the residual stream
        {"name": "combine_8192x4096_top4", "kind": "combine", "rows": 8192, "experts": 64, "top": 4, "out": 4096,
         "residual": True, "dtype": "bfloat16"},
        # one token through its four experts' up projections: the weights' bytes and the launch count
        {"name": "experts_int4_1x2816x4096_64top4", "kind": "experts", "rows": 1, "experts": 64, "top": 4, "out": 2816,
         "in": 4096, "bits": 4, "asym": True, "bias": False, "gather": True, "dtype": "bfloat16"},
        # down projections of some hundred tokens, odd sizes everywhere, INT8 weights with zero-points and a bias
        {"name": "experts_int8_201x1000x2901_10top3", "kind": "experts", "rows": 201, "experts": 10, "top": 3,
         "out": 1000, "in": 2901, "bits": 8, "asym": True, "bias": True, "gather": False, "dtype": "float16"},
        # many requests' single tokens in one batch: every expert's weights are read for about 32 rows
        {"name": "experts_int4_512x2816x4096_64top4", "kind": "experts", "rows": 512, "experts": 64, "top": 4,
         "out": 2816, "in": 4096, "bits": 4, "asym": True, "bias": False, "gather": True, "dtype": "bfloat16"},
        # a long prompt through the up projections of 32 experts: the matrix cores count
        {"name": "experts_int4_8192x2816x4096_32top4", "kind": "experts", "rows": 8192, "experts": 32, "top": 4,
         "out": 2816, "in": 4096, "bits": 4, "asym": True, "bias": False, "gather": True, "dtype": "bfloat16"},
        # one request's token with its adapter
        {"name": "adapters_int4_1x4096x4096_r16", "kind": "adapters", "rows": 1, "out": 4096, "in": 4096, "adapters": 8,
         "rank": 16, "bits": 4, "asym": True, "bias": False, "dtype": "bfloat16"},
        # single tokens of many requests, most with adapters of their own, in an up projection
        {"name": "adapters_int4_64x12288x4096_r16", "kind": "adapters", "rows": 64, "out": 12288, "in": 4096,
         "adapters": 48, "rank": 16, "bits": 4, "asym": True, "bias": False, "dtype": "bfloat16"},
        # a few hundred rows, odd sizes everywhere, INT8 weights with zero-points and a bias
        {"name": "adapters_int8_333x1000x2901_r12", "kind": "adapters", "rows": 333, "out": 1000, "in": 2901,
         "adapters": 5, "rank": 12, "bits": 8, "asym": True, "bias": True, "dtype": "float16"},
        # prompts of a few requests through a down projection, wide adapters
        {"name": "adapters_int4_8192x4096x12288_r64", "kind": "adapters", "rows": 8192, "out": 4096, "in": 12288,
         "adapters": 6, "rank": 64, "bits": 4, "asym": True, "bias": False, "dtype": "bfloat16"},
    ]


def _size(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi]: as it falls, or a multiple of 64."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return min(hi, max(lo, n if rng.random() < 0.5 or n < 64 else n // 64 * 64))


def draw(rng):
    kind = rng.choice(["route", "combine", "experts", "experts", "experts", "adapters", "adapters", "adapters"])
    case = {"kind": kind, "rows": _size(rng, 1, 8192), "dtype": rng.choice(["bfloat16", "bfloat16", "float16", "float32"])}
    if kind != "adapters":
        case["experts"] = _size(rng, 4, 256)
        case["top"] = min(case["experts"], rng.choice([1, 2, 3, 4, 6, 8]))
    if kind == "route":
        case["renormalize"] = rng.random() < 0.5
        case["padded"] = rng.choice([0.0, 0.0, 0.3])
        return case
    case["out"] = _size(rng, 64, 4096 if kind == "combine" else 12288)
    if kind == "combine":
        case["residual"] = rng.random() < 0.5
        while case["rows"] * case["top"] > 8192 * 4:
            case["rows"] //= 2
        return case
    case["in"] = _size(rng, 64, 12288)
    case["bits"] = rng.choice([4, 4, 8])
    case["asym"] = rng.random() < 0.6
    case["bias"] = rng.random() < 0.4
    if kind == "experts":
        case["gather"] = rng.random() < 0.5
        while case["experts"] * case["out"] * case["in"] > 64 * 2816 * 4096:
            case["experts"] = max(1, case["experts"] // 2)
            case["top"] = min(case["top"], case["experts"])
        while case["rows"] * case["top"] * case["out"] * case["in"] > 8192 * 4 * 2816 * 4096:
            case["rows"] = max(1, case["rows"] // 2)
    else:
        case["adapters"], case["rank"] = _size(rng, 1, 64), rng.choice([4, 8, 12, 16, 16, 32, 64, 128])
        if case["dtype"] == "float32":                   # adapters are kept in 16 bits
            case["dtype"] = "bfloat16"
        while case["rows"] * case["out"] * case["in"] > 8192 * 4096 * 12288:
            case["rows"] = max(1, case["rows"] // 2)
    return case


# ---------------------------------------------------------------- inputs

def _rhaz(x):
    return torch.trunc(x + torch.copysign(torch.full_like(x, 0.5), x))


def _stored_weight(g, n, k, bits, asym):
    """Round-to-nearest weights as the converter stores them: codes (INT4: two to a byte, low nibble first), fp16
    scales and int8 zero-points [n, 1]."""
    w = torch.randn(n, k, generator=g, device="cuda") * 0.02
    lo, hi = (-8, 7) if bits == 4 else (-128, 127)
    if asym:
        top, low = w.amax(1, keepdim=True), w.amin(1, keepdim=True)
        s = ((top - low) / (hi - lo)).clamp(min=1e-5).half()
        z = (lo - _rhaz(low / s.float())).clamp(lo, hi)
    else:
        s = (w.abs().amax(1, keepdim=True) / hi).clamp(min=1e-5).half()
        z = None
    q = _rhaz(w / s.float() + (z if z is not None else 0)).clamp(lo, hi).to(torch.int8)
    if bits == 4:
        u = torch.nn.functional.pad(q, (0, q.shape[1] % 2)).view(torch.uint8) & 15
        q = u[:, 0::2] | (u[:, 1::2] << 4)
    return q, s, None if z is None else z.to(torch.int8)


def _codes(g, rows, n):
    """8-bit activations with a scale a row, of normal values with a few louder channels."""
    x = torch.randn(rows, n, generator=g, device="cuda")
    x = x * torch.where(torch.rand(n, generator=g, device="cuda") < 0.01, 8.0, 1.0)
    s = x.abs().amax(1) / 127
    return _rhaz(x / s[:, None]).clamp(-127, 127).to(torch.int8), s


def _logits(g, case):
    """A router's outputs, some experts more in demand than others."""
    popular = 0.5 * torch.randn(case["experts"], generator=g, device="cuda")
    return torch.randn(case["rows"], case["experts"], generator=g, device="cuda") + popular


def _chosen(g, case):
    """(experts int32 [rows, top], weights fp32 [rows, top]) as a router chooses them."""
    top = torch.topk(_logits(g, case), case["top"])
    return top.indices.int(), torch.softmax(top.values, 1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, kind = DTYPES[case["dtype"]], case["kind"]
    state = {"case": case, "dtype": dtype}
    if kind == "route":
        logits = _logits(g, case)
        if case["padded"]:
            logits[torch.rand(case["rows"], generator=g, device="cuda") < case["padded"]] = -math.inf
        state["logits"] = logits.to(dtype)
        return state
    if kind in ("combine", "experts"):
        state["ids"], state["weights"] = _chosen(g, case)
        flat = state["ids"].reshape(-1).long()
        state["order"] = torch.argsort(flat, stable=True)                  # pairs (token * top + choice) by expert
        state["position"] = torch.argsort(state["order"]).reshape(case["rows"], case["top"])
    if kind == "combine":
        state["y"] = torch.randn(case["rows"] * case["top"], case["out"], generator=g, device="cuda").to(dtype)
        state["residual"] = (torch.randn(case["rows"], case["out"], generator=g, device="cuda") * 4).to(dtype) \
            if case["residual"] else None
    if kind == "experts":
        state["counts"] = torch.bincount(flat, minlength=case["experts"]).tolist()   # the plain form's loop
        pairs = case["rows"] * (1 if case["gather"] else case["top"])
        state["codes"], state["scales"] = _codes(g, pairs, case["in"])
        state["layers"] = [_stored_weight(g, case["out"], case["in"], case["bits"], case["asym"])
                           for _ in range(case["experts"])]
        state["bias"] = torch.randn(case["experts"], case["out"], generator=g, device="cuda").to(dtype) \
            if case["bias"] else None
    if kind == "adapters":
        state["codes"], state["scales"] = _codes(g, case["rows"], case["in"])
        state["layers"] = [_stored_weight(g, case["out"], case["in"], case["bits"], case["asym"])]
        state["bias"] = torch.randn(case["out"], generator=g, device="cuda").to(dtype) if case["bias"] else None
        n, r = case["adapters"], case["rank"]
        state["a"] = (torch.randn(n, r, case["in"], generator=g, device="cuda") / math.sqrt(case["in"])).to(dtype)
        state["b"] = (torch.randn(n, case["out"], r, generator=g, device="cuda") * 0.05).to(dtype)
        state["scaling"] = 0.5 + 1.5 * torch.rand(n, generator=g, device="cuda")
        # long batches hold prompts, whose rows follow one another; an eighth of the requests have no adapter
        run = 1 if case["rows"] <= 256 else -(-case["rows"] // (2 * n + 3))
        requests = torch.randint(0, n, (-(-case["rows"] // run),), generator=g, device="cuda")
        requests[torch.rand(requests.shape[0], generator=g, device="cuda") < 0.125] = -1
        state["ids"] = requests.repeat_interleave(run)[: case["rows"]].int()
    if own:       # what a program keeps: weights and adapters laid out, the batch's order, the activations' handle
        import int_crush_converter_amd as icq
        if kind in ("combine", "experts"):
            state["groups"] = icq.group_rows(state["ids"], case["experts"])
        if kind == "experts":
            state["w"] = icq.ExpertWeight([icq.QuantizedWeight(*layer, in_features=case["in"])
                                           for layer in state["layers"]])
        if kind == "adapters":
            state["w"] = icq.QuantizedWeight(*state["layers"][0], in_features=case["in"])
            state["adapters"] = icq.LowRankAdapters(state["a"], state["b"], state["scaling"])
            state["groups"] = icq.group_rows(state["ids"], case["adapters"])
        if kind in ("experts", "adapters"):
            state["act"] = icq.QuantizedActivations.from_codes(state["codes"], state["scales"])
    return state


# ---------------------------------------------------------------- the plain forms

def _plain_route(state):
    case, x = state["case"], state["logits"].float()
    rows, experts, top = case["rows"], case["experts"], case["top"]
    value, ids = torch.sort(x, dim=1, descending=True, stable=True)       # of equal logits the lowest expert first
    value, ids = value[:, :top], ids[:, :top]
    none = value == -math.inf                                             # what the router's mask took out
    peak = value[:, :1].clamp(min=torch.finfo(torch.float32).min)
    e = torch.exp(value - peak)
    total = e.sum(1, keepdim=True) if case["renormalize"] else torch.exp(x - peak).sum(1, keepdim=True)
    weights = torch.where(none, 0.0, e / total)
    ids = torch.where(none, experts, ids)
    flat = ids.reshape(-1)
    order = torch.argsort(flat, stable=True)
    offsets = torch.searchsorted(flat[order], torch.arange(experts + 1, device=flat.device))
    position = torch.empty_like(order)
    position[order] = torch.arange(rows * top, device=order.device)
    none = none.reshape(-1)
    return {"ids": torch.where(none, -1, flat).reshape(rows, top).int(), "weights": weights, "offsets": offsets.int(),
            "order": torch.where(none[order], -1, order).int(),
            "position": torch.where(none, -1, position).reshape(rows, top).int()}


def _plain_combine(state):
    y = (state["y"].float()[state["position"]] * state["weights"][:, :, None]).sum(1)
    if state["residual"] is not None:
        y = y + state["residual"].float()
    return y.to(state["dtype"])


def _plain_weight(layer, bits, k):
    w, s, z = layer
    if bits == 4:
        u = torch.stack((w & 15, w >> 4), 2).reshape(w.shape[0], -1)[:, :k]
        w = (u ^ 8).to(torch.int8) - 8
    w = w.float()
    return (w if z is None else w - z.float()) * s.float()


def _plain_experts(state):
    case, out, at = state["case"], [], 0
    x = state["codes"].float() * state["scales"][:, None]
    for e, count in enumerate(state["counts"]):
        if count:
            rows = x[state["order"][at: at + count] // case["top"]] if case["gather"] else x[at: at + count]
            y = rows @ _plain_weight(state["layers"][e], case["bits"], case["in"]).T
            out.append(y if state["bias"] is None else y + state["bias"][e].float())
            at += count
    return torch.cat(out).to(state["dtype"])


def _plain_adapters(state):
    case, n, r = state["case"], state["case"]["adapters"], state["case"]["rank"]
    x = state["codes"].float() * state["scales"][:, None]
    y = x @ _plain_weight(state["layers"][0], case["bits"], case["in"]).T
    # all adapters' first factors at once, then the row's own are kept
    t = (x @ state["a"].float().reshape(n * r, -1).T).reshape(-1, n, r)
    t = t * (state["ids"][:, None] == torch.arange(n, device=t.device)).float()[:, :, None] * state["scaling"][:, None]
    y = y + t.reshape(-1, n * r) @ state["b"].float().permute(0, 2, 1).reshape(n * r, -1)
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(state["dtype"])


# ---------------------------------------------------------------- one pass

def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if not own:
        return {"route": _plain_route, "combine": _plain_combine, "experts": _plain_experts,
                "adapters": _plain_adapters}[kind](state)
    import int_crush_converter_amd as icq
    if kind == "route":
        groups, weights = icq.route_tokens(state["logits"], case["top"], renormalize=case["renormalize"])
        return {"ids": groups.ids, "weights": weights, "offsets": groups.offsets, "order": groups.order,
                "position": groups.position}
    if kind == "combine":
        return icq.combine_experts(state["y"], state["groups"], state["weights"], state["residual"])
    if kind == "experts":
        return icq.expert_linear(state["act"], state["w"], state["groups"], state["bias"], gather=case["gather"],
                                 out_dtype=state["dtype"])
    return icq.quantized_linear(state["act"], state["w"], state["bias"], adapters=state["adapters"],
                                groups=state["groups"], out_dtype=state["dtype"])


def _expected(n, draws):
    """How many of n are met by so many draws, each as likely as the next."""
    return n * (1 - (1 - 1 / n) ** draws)


def work(case):
    """What one pass cannot do without: its inputs read once and its outputs written once, the weights of the experts
    and adapters that its rows meet, and the multiplications and additions of its definition."""
    m, kind = case["rows"], case["kind"]
    size = 4 if case["dtype"] == "float32" else 2
    if kind == "route":
        e, top = case["experts"], case["top"]
        return {"bytes": size * m * e + 16 * m * top + 4 * (e + 1), "flops": 4 * m * e}
    n = case["out"]
    if kind == "combine":
        pairs = m * case["top"]
        return {"bytes": size * (pairs + m * (2 if case["residual"] else 1)) * n + 8 * pairs, "flops": 2 * pairs * n}
    k = case["in"]
    layer = n * -(-k * case["bits"] // 8) + n * (3 if case["asym"] else 2) + (size * n if case["bias"] else 0)
    if kind == "experts":
        pairs, e = m * case["top"], case["experts"]
        met = e * (1 - (1 - case["top"] / e) ** m)         # a token's choices differ
        read = m if case["gather"] else pairs
        return {"bytes": met * layer + read * (k + 4) + size * pairs * n, "flops": 2 * pairs * n * k}
    r = case["rank"]
    met = _expected(case["adapters"], m * 0.875 if m <= 256 else 0.875 * (2 * case["adapters"] + 3))
    return {"bytes": layer + m * (k + 4) + size * m * n + met * size * r * (n + k),
            "flops": 2 * m * n * k + 0.875 * 2 * m * r * (n + k)}


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_route(state):
    case, x = state["case"], state["logits"].double()
    rows, experts, top = case["rows"], case["experts"], case["top"]
    left, ids, value = x.clone(), [], []
    number = torch.arange(experts, device=x.device)
    for _ in range(top):                                                   # the largest left, the lowest of equals
        best = left.max(1, keepdim=True).values
        first = torch.where(left == best, number, experts).min(1, keepdim=True).values
        ids.append(torch.where(best == -math.inf, -1, first))
        value.append(best)
        left.scatter_(1, first, -math.inf)
    ids, value = torch.cat(ids, 1), torch.cat(value, 1)
    share = value if case["renormalize"] else x
    weights = (value - torch.logsumexp(share, 1, keepdim=True)).exp()
    weights = torch.where(ids < 0, 0.0, weights)
    flat, at = ids.reshape(-1), 0
    order, position = torch.full_like(flat, -1), torch.full_like(flat, -1)
    offsets = [0]
    for e in range(experts):
        mine = (flat == e).nonzero()[:, 0]
        order[at: at + mine.shape[0]] = mine
        position[mine] = at + torch.arange(mine.shape[0], device=flat.device)
        at += mine.shape[0]
        offsets.append(at)
    return {"ids": ids.int(), "weights": weights, "offsets": torch.tensor(offsets, dtype=torch.int32, device=x.device),
            "order": order.int(), "position": position.reshape(rows, top).int()}


def _exact_combine(state):
    case = state["case"]
    y = torch.zeros(case["rows"], case["out"], dtype=torch.float64, device="cuda") if state["residual"] is None \
        else state["residual"].double()
    for j in range(case["top"]):
        y = y + state["weights"][:, j: j + 1].double() * state["y"][state["position"][:, j]].double()
    return y


def _exact_layer(layer, bits, k):
    w, s, z = layer
    if bits == 4:
        both = torch.empty(w.shape[0], w.shape[1] * 2, dtype=torch.float64, device=w.device)
        both[:, ::2], both[:, 1::2] = (w % 16).double(), (w // 16).double()
        w = torch.where(both > 7, both - 16, both)[:, :k]
    w = w.double()
    return s.double() * (w if z is None else w - z.double())


def _exact_experts(state):
    case = state["case"]
    x = state["codes"].double() * state["scales"].double()[:, None]
    y = torch.empty(case["rows"] * case["top"], case["out"], dtype=torch.float64, device="cuda")
    pair_expert = state["ids"].reshape(-1)
    for e in range(case["experts"]):
        pairs = (pair_expert == e).nonzero()[:, 0]
        if pairs.shape[0] == 0:
            continue
        at = state["position"].reshape(-1)[pairs]
        rows = x[pairs // case["top"]] if case["gather"] else x[at]
        y[at] = rows @ _exact_layer(state["layers"][e], case["bits"], case["in"]).T \
            + (0 if state["bias"] is None else state["bias"][e].double())
    return y


def _exact_adapters(state):
    case = state["case"]
    x = state["codes"].double() * state["scales"].double()[:, None]
    y = x @ _exact_layer(state["layers"][0], case["bits"], case["in"]).T
    if state["bias"] is not None:
        y += state["bias"].double()
    for n in range(case["adapters"]):
        mine = (state["ids"] == n).nonzero()[:, 0]
        if mine.shape[0]:
            y[mine] += state["scaling"][n].double() * (x[mine] @ state["a"][n].double().T) @ state["b"][n].double().T
    return y


def exact(case, seed):
    state = prepare(case, seed)
    return {"route": _exact_route, "combine": _exact_combine, "experts": _exact_experts,
            "adapters": _exact_adapters}[case["kind"]](state)
