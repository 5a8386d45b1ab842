"""The operators that run a quantised layer, as cases that can be timed and compared.

Four operators, each in a plain form (elementary torch operations in 32 bits)
and as the package's own call: the root-mean-square norm with the residual's
addition and the rotation whose output is 8-bit activations with a scale for
each token; the product of such activations with the INT4 / INT8 weights that
the converter stores; the quantisation to microscaled 4-bit floating point
(E2M1 elements, one E8M0 scale for 32 of them); and the product of two
operands in that format.  ``exact`` restates each in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EPS = 1e-6
TINY = 1e-30          # the smallest row maximum that an activation scale stands for
BLOCK = 32            # elements that share one E8M0 scale


def listed():
    return [
        # one token on its way into a layer: launches and latency count
        {"name": "norm_rot256_1x4096", "kind": "norm", "rows": 1, "in": 4096, "rot": 256, "residual": True,
         "dtype": "bfloat16"},
        # an odd number of tokens and a width that is no multiple of the rotation, the first norm of a model
        {"name": "norm_rot64_777x2901", "kind": "norm", "rows": 777, "in": 2901, "rot": 64, "residual": False,
         "dtype": "float16"},
        # a long prompt through the norm before a projection
        {"name": "norm_rot256_8192x4096", "kind": "norm", "rows": 8192, "in": 4096, "rot": 256, "residual": True,
         "dtype": "bfloat16"},
        # the input of a down projection, which no norm precedes, not rotated, for a long prompt
        {"name": "quantize_8192x12288", "kind": "quantize", "rows": 8192, "in": 12288, "rot": 0, "dtype": "bfloat16"},
        # one token through an up projection with the converter's default weights: the weights' bytes count
        {"name": "linear_int4_1x12288x4096", "kind": "linear", "rows": 1, "out": 12288, "in": 4096, "bits": 4,
         "asym": True, "bias": False, "dtype": "bfloat16"},
        # a few hundred tokens, odd sizes everywhere, INT8 weights with zero-points and a bias
        {"name": "linear_int8_333x1000x2901", "kind": "linear", "rows": 333, "out": 1000, "in": 2901, "bits": 8,
         "asym": True, "bias": True, "dtype": "float16"},
        # a long prompt through a down projection: the matrix cores count
        {"name": "linear_int4_8192x4096x12288", "kind": "linear", "rows": 8192, "out": 4096, "in": 12288, "bits": 4,
         "asym": True, "bias": False, "dtype": "bfloat16"},
        # weights of an odd layer, once for each layer of a model
        {"name": "mxfp4_quantize_5000x2900", "kind": "mxquantize", "rows": 5000, "in": 2900, "dtype": "float16"},
        # the activations of a long prompt
        {"name": "mxfp4_quantize_8192x12288", "kind": "mxquantize", "rows": 8192, "in": 12288, "dtype": "bfloat16"},
        # a small batch of single tokens through a down projection
        {"name": "mxfp4_linear_8x4096x12288", "kind": "mxlinear", "rows": 8, "out": 4096, "in": 12288, "bias": False,
         "dtype": "bfloat16"},
        # a prompt of odd length, sizes that are no multiple of any tile
        {"name": "mxfp4_linear_701x5000x2900", "kind": "mxlinear", "rows": 701, "out": 5000, "in": 2900, "bias": True,
         "dtype": "float32"},
        # a long prompt through an up projection
        {"name": "mxfp4_linear_8192x12288x4096", "kind": "mxlinear", "rows": 8192, "out": 12288, "in": 4096,
         "bias": False, "dtype": "bfloat16"},
    ]


def _size(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi]: as it falls, or a multiple of 64."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return min(hi, max(lo, n if rng.random() < 0.5 or n < 64 else n // 64 * 64))


def draw(rng):
    kind = rng.choice(["norm", "quantize", "linear", "linear", "mxquantize", "mxlinear", "mxlinear"])
    case = {"kind": kind, "rows": _size(rng, 1, 8192), "in": _size(rng, 64, 12288),
            "dtype": rng.choice(["bfloat16", "bfloat16", "float16", "float32"])}
    if kind in ("norm", "quantize"):
        case["rot"] = rng.choice([0, 16, 64, 256, 256])
        if kind == "norm":
            case["residual"] = rng.random() < 0.7
    if kind in ("linear", "mxlinear"):
        case["out"] = _size(rng, 64, 12288)
        while case["rows"] * case["out"] * case["in"] > 8192 * 12288 * 4096:
            case["rows"] = max(1, case["rows"] // 2)
        case["bias"] = rng.random() < 0.5
        if kind == "linear":
            case["bits"] = rng.choice([4, 4, 8])
            case["asym"] = rng.random() < 0.6
    return case


# ---------------------------------------------------------------- inputs

def _activations(g, rows, n, dtype):
    """Normal values with a few louder channels, as a residual stream has them."""
    x = torch.randn(rows, n, generator=g, device="cuda")
    loud = torch.rand(n, generator=g, device="cuda") < 0.01
    return (x * torch.where(loud, 8.0, 1.0)).to(dtype)


def _rhaz(x):
    return torch.trunc(x + torch.copysign(torch.full_like(x, 0.5), x))


def _stored_weight(g, case):
    """Round-to-nearest weights as the converter stores them: codes (INT4: two to a byte, low nibble first),
    fp16 scales and int8 zero-points [out, 1]."""
    w = torch.randn(case["out"], case["in"], generator=g, device="cuda") * 0.02
    lo, hi = (-8, 7) if case["bits"] == 4 else (-128, 127)
    if case["asym"]:
        top, low = w.amax(1, keepdim=True), w.amin(1, keepdim=True)
        s = ((top - low) / (hi - lo)).clamp(min=1e-5).half()
        z = (lo - _rhaz(low / s.float())).clamp(lo, hi)
    else:
        s = (w.abs().amax(1, keepdim=True) / hi).clamp(min=1e-5).half()
        z = None
    q = _rhaz(w / s.float() + (z if z is not None else 0)).clamp(lo, hi).to(torch.int8)
    if case["bits"] == 4:
        u = torch.nn.functional.pad(q, (0, q.shape[1] % 2)).view(torch.uint8) & 15
        q = u[:, 0::2] | (u[:, 1::2] << 4)
    return q, s, None if z is None else z.to(torch.int8)


def _mx_parts(x):
    """(elements, exponents): E2M1 values in fp32 [rows, blocks, 32] and the power-of-two exponent of each block."""
    rows, n = x.shape
    b = torch.nn.functional.pad(x.float(), (0, -n % BLOCK)).reshape(rows, -1, BLOCK)
    top = b.abs().amax(2, keepdim=True)
    e = (torch.frexp(top)[1] - 3).clamp(-127, 127)             # floor(log2(top)) - 2: E2M1 reaches 1.5 * 2^2
    e = torch.where(top > 0, e, -127)
    v = torch.ldexp(b, -e)
    a = v.abs().clamp(max=6.0)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.copysign(torch.round(a / step) * step, v), e


def _mx_packed(x):
    """An operand in microscaled 4-bit form: uint8 [rows, blocks * 16] (even element in the low nibble) and E8M0
    bytes [rows, blocks]."""
    v, e = _mx_parts(x)
    a = v.abs()
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = (code | (torch.signbit(v).to(torch.uint8) << 3)).reshape(x.shape[0], -1)
    return code[:, 0::2] | (code[:, 1::2] << 4), (e[:, :, 0] + 127).to(torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, kind, n = DTYPES[case["dtype"]], case["kind"], case["in"]
    state = {"case": case, "dtype": dtype}
    if kind in ("norm", "quantize", "mxquantize"):
        state["x"] = _activations(g, case["rows"], n, dtype)
        if kind == "norm":
            state["weight"] = (1 + 0.1 * torch.randn(n, generator=g, device="cuda")).to(dtype)
            state["residual"] = _activations(g, case["rows"], n, dtype) * 2 if case["residual"] else None
        return state
    state["bias"] = torch.randn(case["out"], generator=g, device="cuda").to(dtype) if case["bias"] else None
    x = _activations(g, case["rows"], n, torch.float32)
    if kind == "linear":
        s = x.abs().amax(1) / 127
        state["codes"], state["scales"] = _rhaz(x / s[:, None]).clamp(-127, 127).to(torch.int8), s
        state["stored"], state["wscales"], state["zeros"] = _stored_weight(g, case)
    else:
        state["codes"], state["scales"] = _mx_packed(x)
        w = torch.randn(case["out"], n, generator=g, device="cuda") * 0.02
        state["stored"], state["wscales"] = _mx_packed(w)
    if own:                # what a program keeps from load to load: the weights laid out, the activations' handle
        import int_crush_converter_amd as icq
        if kind == "linear":
            state["act"] = icq.QuantizedActivations.from_codes(state["codes"], state["scales"])
            state["w"] = icq.QuantizedWeight(state["stored"], state["wscales"], state["zeros"], in_features=n)
        else:
            state["act"] = icq.Mxfp4Tensor.from_packed(state["codes"], state["scales"], in_features=n)
            state["w"] = icq.Mxfp4Tensor.from_packed(state["stored"], state["wscales"], in_features=n)
    return state


# ---------------------------------------------------------------- the plain forms

def _hadamard(rot):
    """The regular Hadamard matrix (H4 / 2) kron ... kron (H4 / 2) of order rot."""
    h4 = torch.tensor([[1, 1, 1, -1], [1, 1, -1, 1], [1, -1, 1, 1], [-1, 1, 1, 1]], dtype=torch.float32,
                      device="cuda") / 2
    h = h4
    while h.shape[0] < rot:
        h = torch.kron(h, h4)
    return h


def _plain_quantize(y, rot):
    """Rotated (padded) rows as the values of their 8-bit codes: q * s, s = max|y| / 127."""
    if rot:
        y = torch.nn.functional.pad(y, (0, -y.shape[1] % rot))
        y = (y.reshape(-1, rot) @ _hadamard(rot).T).reshape(y.shape)
    top = y.abs().amax(1, keepdim=True).clamp(min=TINY)
    return (_rhaz(y * (127 / top)).clamp(-127, 127) * (top / 127)).to(torch.bfloat16)


def _plain_norm(state):
    case = state["case"]
    h = state["x"].float()
    if state["residual"] is not None:
        h = h + state["residual"].float()
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * state["weight"].float()
    out = {"values": _plain_quantize(y, case["rot"])}
    if state["residual"] is not None:
        out["residual"] = h.to(state["dtype"])
    return out


def _plain_linear(state):
    case = state["case"]
    w = state["stored"]
    if case["bits"] == 4:
        u = torch.stack((w & 15, w >> 4), 2).reshape(case["out"], -1)[:, : case["in"]]
        w = ((u ^ 8).to(torch.int8) - 8)
    w = w.float()
    if state["zeros"] is not None:
        w = w - state["zeros"].float()
    y = (state["codes"].float() * state["scales"][:, None]) @ (w * state["wscales"].float()).T
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(state["dtype"])


def _plain_mx_values(codes, scales, n):
    u = torch.stack((codes & 15, codes >> 4), 2).reshape(codes.shape[0], -1)
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    v = table[u.int()].reshape(codes.shape[0], -1, BLOCK)
    return torch.ldexp(v, scales.int()[:, :, None] - 127).reshape(codes.shape[0], -1)[:, :n]


def _plain_mx_linear(state):
    n = state["case"]["in"]
    y = _plain_mx_values(state["codes"], state["scales"], n) @ _plain_mx_values(state["stored"], state["wscales"], n).T
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(state["dtype"])


def _plain_mx_quantize(state):
    v, e = _mx_parts(state["x"])
    return torch.ldexp(v, e).reshape(v.shape[0], -1)[:, : state["case"]["in"]].to(torch.bfloat16)


# ---------------------------------------------------------------- one pass

def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if not own:
        if kind == "norm":
            return _plain_norm(state)
        if kind == "quantize":
            return {"values": _plain_quantize(state["x"].float(), case["rot"])}
        if kind == "linear":
            return _plain_linear(state)
        return _plain_mx_quantize(state) if kind == "mxquantize" else _plain_mx_linear(state)
    import int_crush_converter_amd as icq
    if kind == "norm":
        q, residual = icq.rms_norm_quantize(state["x"], state["weight"], state["residual"], eps=EPS,
                                            rot_size=case["rot"])
        out = {"values": q.dequantize(torch.bfloat16)}
        if residual is not None:
            out["residual"] = residual
        return out
    if kind == "quantize":
        return {"values": icq.quantize_activations(state["x"], rot_size=case["rot"]).dequantize(torch.bfloat16)}
    if kind == "linear":
        return icq.quantized_linear(state["act"], state["w"], state["bias"], out_dtype=state["dtype"])
    if kind == "mxquantize":
        return icq.mxfp4_quantize(state["x"]).dequantize(torch.bfloat16)
    return icq.mxfp4_linear(state["act"], state["w"], state["bias"], out_dtype=state["dtype"])


def work(case):
    """What one pass cannot do without: its inputs read once and its outputs written once, and the multiplications
    and additions of its definition."""
    m, k, kind = case["rows"], case["in"], case["kind"]
    size = 4 if case["dtype"] == "float32" else 2
    if kind in ("norm", "quantize"):
        kp = k + (-k % case["rot"] if case["rot"] else 0)
        stream = size * m * k * (3 if case.get("residual") else 1) + (size * k if kind == "norm" else 0)
        stages = 3 * round(math.log(case["rot"], 4)) if case["rot"] else 0
        return {"bytes": stream + 2 * m * kp, "flops": m * k * (5 if kind == "norm" else 0) + m * kp * (stages + 3)}
    if kind == "mxquantize":
        return {"bytes": (size + 2) * m * k, "flops": 3 * m * k}
    n = case["out"]
    bias = size * n if case["bias"] else 0
    if kind == "linear":
        weights = n * -(-k * case["bits"] // 8) + n * (3 if case["asym"] else 2)
        return {"bytes": m * k + 4 * m + weights + bias + size * m * n, "flops": 2 * m * n * k}
    blocks = -(-k // BLOCK)
    return {"bytes": 17 * blocks * (m + n) + bias + size * m * n, "flops": 2 * m * n * k}


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_rotate(y, rot):
    """The rotation digit by digit: y_d = (x_0 + x_1 + x_2 + x_3) / 2 - x_(3 - d) for each base-4 digit d."""
    rows, n = y.shape
    y = torch.cat((y, y.new_zeros(rows, -n % rot)), 1)
    width = y.shape[1]
    digit = 1
    while digit < rot:
        v = y.reshape(-1, 4, digit)
        y = (v.sum(1, keepdim=True) / 2 - v.flip(1)).reshape(rows, width)
        digit *= 4
    return y


def _exact_codes(y):
    """The values of the 8-bit codes, halves away from zero, in 64 bits."""
    s = y.abs().max(1, keepdim=True).values.clamp(min=TINY) / 127
    t = y / s
    return t.sign() * (t.abs() + 0.5).floor().clamp(max=127) * s


def _exact_e2m1(x):
    """Each block's values in the format, the nearest of the eight magnitudes, ties to the even code."""
    rows, n = x.shape
    out = torch.empty(rows, n, dtype=torch.float64, device=x.device)
    grid = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    for at in range(0, rows, 2048):
        b = torch.nn.functional.pad(x[at: at + 2048].double(), (0, -n % BLOCK)).unflatten(1, (-1, BLOCK))
        top = b.abs().max(2, keepdim=True).values
        scale = torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -125))) - 2).clamp(min=2.0 ** -127)
        a, v = b.abs() / scale, torch.zeros_like(b)
        for i in range(1, 8):
            edge = (grid[i - 1] + grid[i]) / 2
            v = torch.where(a > edge if i % 2 else a >= edge, grid[i], v)
        out[at: at + 2048] = (v * scale * b.sign()).flatten(1)[:, :n]
    return out


def _exact_nibbles(packed, n):
    both = torch.empty(packed.shape[0], packed.shape[1] * 2, dtype=torch.long, device=packed.device)
    both[:, ::2], both[:, 1::2] = packed.long() % 16, packed.long() // 16
    return both[:, :n]


def _exact_mx_operand(codes, scales, n):
    u = _exact_nibbles(codes, n)
    e, m = (u % 8) // 2, u % 2
    a = torch.where(e == 0, m / 2, (1 + m.double() / 2) * torch.exp2((e - 1).double()))
    s = torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, 1)[:, :n]
    return torch.where(u >= 8, -a, a).double() * s


def exact(case, seed):
    state, kind = prepare(case, seed), case["kind"]
    n = case["in"]
    if kind in ("norm", "quantize"):
        y, out = state["x"].double(), {}
        if kind == "norm":
            if state["residual"] is not None:
                y = y + state["residual"].double()
                out["residual"] = y
            y = y / torch.sqrt(y.square().sum(1, keepdim=True) / n + EPS) * state["weight"].double()
        out["values"] = _exact_codes(_exact_rotate(y, case["rot"]) if case["rot"] else y)
        return out
    if kind == "mxquantize":
        return _exact_e2m1(state["x"])
    if kind == "linear":
        a = state["codes"].double() * state["scales"].double()[:, None]
        w = state["stored"].double()
        if case["bits"] == 4:
            w = _exact_nibbles(state["stored"], n).double()
            w = torch.where(w > 7, w - 16, w)
        if state["zeros"] is not None:
            w = w - state["zeros"].double()
        w = w * state["wscales"].double()
    else:
        a = _exact_mx_operand(state["codes"], state["scales"], n)
        w = _exact_mx_operand(state["stored"], state["wscales"], n)
    y = a @ w.T
    return y if state["bias"] is None else y + state["bias"].double()
