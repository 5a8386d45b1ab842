"""8-bit activation codes where the quotient is a half, against integers.

With the row's values and its largest magnitude b as integers (times a power
of two) the code of a is sign(a) floor((254 |a| + b) / (2 b)), exactly.  16-bit
values that are neither rotated nor normalised lie at least 2^-19 of their
quotient from a half that they do not reach, far more than the kernel's own
rounding, so all their codes are compared; of fp32 and rotated rows those that
are halves.
"""

from __future__ import annotations

import pytest
import torch

from oracle import torch_ref as ref

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def integer_codes(a):
    b = a.abs().amax(1, keepdim=True)
    return a.sign() * ((254 * a.abs() + b) // (2 * b))


def halves(rows, K, t_max, seed):
    """Integer rows: a maximum of 254 t and multiples (2 k + 1) t, whose quotients are k + 1/2."""
    g = torch.Generator().manual_seed(seed)
    t = torch.randint(1, t_max + 1, (rows, 1), generator=g)
    a = (2 * torch.randint(0, 127, (rows, K), generator=g) + 1) * t * (1 - 2 * torch.randint(0, 2, (rows, K), generator=g))
    a[:, K // 2] = 254 * t[:, 0]
    return a


@pytest.mark.parametrize("K", [2, 200, 4096, 17000])
@pytest.mark.parametrize("dtype,bits", [(BF16, 8), (F16, 11)])
def test_every_code_of_16_bit_rows(gpu_dev, K, dtype, bits):
    import int_crush_converter_amd as icq
    g = torch.Generator().manual_seed(K)
    rows = 1 << (bits - 1)                                         # a maximum of every mantissa
    top = torch.arange(1 << (bits - 1), 1 << bits)[:, None]
    a = (torch.rand(rows, K, generator=g) * (top + 1)).long().clamp(max=(1 << bits) - 1)
    a = torch.minimum(a, top) * (1 - 2 * torch.randint(0, 2, (rows, K), generator=g))
    a[:, ::2] *= 2
    a[:, 0] = 2 * top[:, 0]
    a[:, 1] = -top[:, 0]                                           # a half wherever its maximum's factor rounds
    for shift in (0, -20, 4):
        x = torch.ldexp(a.double(), torch.tensor(shift))
        assert torch.equal(x.to(dtype).double(), x)
        assert torch.equal(icq.quantize_activations(x.to(dtype).to(gpu_dev)).codes.cpu().long(), integer_codes(a))


@pytest.mark.parametrize("K", [3, 129, 4100, 16640])
@pytest.mark.parametrize("dtype,t_max", [(F16, 8), (F32, 60000)])
def test_halves_round_away(gpu_dev, K, dtype, t_max):
    import int_crush_converter_amd as icq
    a = halves(300, K, t_max, K)
    q = icq.quantize_activations(a.to(dtype).to(gpu_dev)).codes.cpu().long()
    assert torch.equal(a.to(dtype).long(), a) and torch.equal(q, integer_codes(a))


@pytest.mark.parametrize("rot", [4, 16, 64, 256])
def test_halves_of_rotated_rows(gpu_dev, rot):
    """Rows whose rotation is a row of integers, formed exactly: every partial sum has fewer than 24 bits."""
    import int_crush_converter_amd as icq
    a = halves(200, 2 * rot, 9, rot)
    x = (a.double().reshape(200, -1, rot) @ ref.hadamard_regular(rot, torch.float64)).reshape(200, -1)
    assert torch.equal(x.float().double(), x)
    q = icq.quantize_activations(x.float().to(gpu_dev), rot_size=rot).codes.cpu().long()
    assert torch.equal(q, integer_codes(a))


@pytest.mark.parametrize("seed,k", [(433, 120), (3110, 123)])
def test_a_row_has_one_norm(gpu_dev, seed, k):
    """Equal values anywhere in a row have equal codes: rows whose sum of squares rounds differently in other orders,
    with a value next to a half in the first column of four groups of lanes."""
    import numpy as np
    import int_crush_converter_amd as icq
    K = 1024
    r = np.random.RandomState(seed)
    x = torch.from_numpy((r.randint(-512, 513, K) / 256).astype(np.float32))
    x[500] = 6.0
    near = np.float32((k + 0.5) * 6 / 127)
    for step in range(-2, 3):
        c = near
        for _ in range(abs(step)):
            c = np.nextafter(c, np.float32(np.sign(step) * 100))
        x[[0, 64, 128, 192]] = float(c)
        q, _ = icq.rms_norm_quantize(x[None].to(gpu_dev), torch.ones(K, device=gpu_dev))
        assert q.codes[0, [0, 64, 128, 192]].unique().numel() == 1
