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


def test_sizes_reach_every_form(gpu_dev):
    import int_crush_converter_amd._native as nat
    assert {(nat.lib().ic_linear_form(k, m, n), d >= 4096) for m, n, d, _, _, _ in EXACT for k in (0, 1)} >= {(0, False), (128, False), (256, False), (256, True)}
