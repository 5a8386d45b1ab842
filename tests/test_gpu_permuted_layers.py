"""Products with layers that the converter permuted: the file's codes with
their columns put back in order, against 64 bits (the bound of the integer
products: fp32 results within 2^-21 of |y|)."""

from __future__ import annotations

import pytest
import torch
from safetensors.torch import load_file, save_file

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("rot,asym", [(256, True), (64, False)])
def test_permuted_file(gpu_dev, tmp_path, bits, rot, asym):
    """A file written with the permutation accepted for every layer, run from its stored tensors."""
    import int_crush_converter_amd as icq
    from int_crush_converter_amd import packing
    g = torch.Generator().manual_seed(bits + rot)
    shapes = {"a.weight": (96, 512), "b.weight": (130, 300), "c.weight": (33, 1024)}
    state = {n: (torch.randn(s, generator=g) * torch.exp(torch.randn(s[1], generator=g)) * 0.02).to(BF16) for n, s in shapes.items()}
    src = str(tmp_path / "in.safetensors")
    save_file(state, src)
    icq.quantize_model(icq.QuantizeConfig(input_path=src, output_dir=str(tmp_path / "out"), rot_size=rot, int_bits=bits,
                                          asymmetric=asym, use_permuquant=True, tau=-1.0))
    stored = load_file(str(tmp_path / "out" / "model.safetensors"))
    for n, (N, K) in shapes.items():
        Kp, perm = -(-K // rot) * rot, stored[f"{n}_perm"].long()
        assert perm.numel() == K and not torch.equal(perm, torch.arange(K))
        s, z = stored[f"{n}_scale"], stored.get(f"{n}_zp")
        w = icq.QuantizedWeight(stored[n], s, z, permutation=stored[f"{n}_perm"], in_features=Kp)
        x = torch.randn(20, K, generator=g).to(BF16)
        q = icq.quantize_activations(x.to(gpu_dev), rot_size=rot)
        y = icq.quantized_linear(q, w, out_dtype=F32).cpu().double()
        # the definition: the activations' columns in the stored order
        codes = stored[n] if bits == 8 else packing.unpack_int4(stored[n].to(gpu_dev), Kp).cpu()
        w64 = codes.double() - (0 if z is None else z.double().reshape(N, 1))
        a64 = q.codes.cpu().double()
        a64[:, :K] = a64[:, perm]
        want = (a64 @ w64.T) * q.scales.cpu().double()[:, None] * s.double().reshape(1, N)
        assert ((y - want).abs() <= 2.0 ** -21 * want.abs() + 1e-12).all()
        # and near the layer that was converted
        ideal = x.double() @ state[n].double().T
        assert (y - ideal).norm() / ideal.norm() < (0.3 if bits == 4 else 0.04)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("N,K,n", [(1, 2, 2), (17, 129, 129), (40, 256, 200), (5, 77, 1), (6, 64, 0)])
def test_partial_permutations(gpu_dev, bits, N, K, n):
    """Permutations of the first n columns, odd rows of nibbles, either integer type, host or GPU, equal the same weight
    stored in order."""
    import int_crush_converter_amd as icq
    g = torch.Generator().manual_seed(N + K)
    lo, hi = (-8, 8) if bits == 4 else (-128, 128)
    q = torch.randint(lo, hi, (N, K), generator=g).to(torch.int8)
    perm = torch.randperm(n, generator=g)
    p = q.clone()
    p[:, :n] = q[:, perm]
    store = lambda t: icq.packing.pack_int4(t.to(gpu_dev)) if bits == 4 else t.to(gpu_dev)       # noqa: E731
    s = torch.rand(N, generator=g)
    plain = icq.QuantizedWeight(store(q), s, in_features=K)
    for pt in (perm, perm.to(torch.int32), perm.to(gpu_dev)):
        assert torch.equal(icq.QuantizedWeight(store(p), s, permutation=pt, in_features=K).tiles, plain.tiles)


def test_refusals(gpu_dev):
    import int_crush_converter_amd as icq
    q, s = torch.zeros(4, 64, dtype=torch.int8, device=gpu_dev), torch.ones(4)
    for bad in (torch.arange(65), torch.zeros(3, dtype=torch.int64), torch.tensor([1, 2]), torch.tensor([-1, 0])):
        with pytest.raises(ValueError, match="permutation"):
            icq.QuantizedWeight(q, s, permutation=bad)
    for bad in (torch.arange(64).float(), torch.arange(64).reshape(8, 8)):
        with pytest.raises(ValueError, match="expected a permutation"):
            icq.QuantizedWeight(q, s, permutation=bad)
