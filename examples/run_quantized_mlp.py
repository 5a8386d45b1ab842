"""A gated feed-forward block, converted to a file and run from it.

The block  y = x + W_down (silu(W_gate n) * (W_up n)),  n = norm(x)  with
random weights is quantised by ``quantize_model`` (rotation 256) and run in
three ways on the same input: as it was, with INT4 or INT8 weights and 8-bit
activations (norm, rotation and quantisation in one pass, integer products),
and in microscaled 4-bit floating point.  Prints how far each is from the
unquantised block, for a prompt and for one token.

    python examples/run_quantized_mlp.py [--hidden 1024] [--inner 2816] [--rows 300]
"""

from __future__ import annotations

import argparse
import os
import sys
import tempfile

import torch
import torch.nn.functional as F
from safetensors.torch import load_file, save_file

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import int_crush_converter_amd as icq  # noqa: E402

ROT = 256
NAMES = ("mlp.gate.weight", "mlp.up.weight", "mlp.down.weight")


def convert(state: dict[str, torch.Tensor], bits: int, folder: str) -> dict[str, icq.QuantizedWeight]:
    """The converter's file for these weights, and its layers laid out for ``quantized_linear``."""
    src = os.path.join(folder, "in.safetensors")
    save_file(state, src)
    out = os.path.join(folder, f"int{bits}")
    icq.quantize_model(icq.QuantizeConfig(input_path=src, output_dir=out, rot_size=ROT, int_bits=bits,
                                          asymmetric=True))
    stored = load_file(os.path.join(out, "model.safetensors"))
    return {n: icq.QuantizedWeight(stored[n], stored[f"{n}_scale"], stored.get(f"{n}_zp"),
                                   permutation=stored.get(f"{n}_perm")) for n in NAMES}


def run_integer(x, residual, gain, w):
    q, h = icq.rms_norm_quantize(x, gain, residual, rot_size=ROT)
    gate, up = icq.quantized_linear(q, w[NAMES[0]]), icq.quantized_linear(q, w[NAMES[1]])
    inner = icq.quantize_activations(F.silu(gate) * up, rot_size=ROT)
    return h + icq.quantized_linear(inner, w[NAMES[2]])


def run_mxfp4(x, residual, gain, w):
    h = x + residual
    n = F.rms_norm(h.float(), (h.shape[-1],), gain.float(), 1e-6)
    q = icq.mxfp4_quantize(icq.rotate_activations(n, ROT))
    gate, up = icq.mxfp4_linear(q, w[NAMES[0]]), icq.mxfp4_linear(q, w[NAMES[1]])
    inner = icq.mxfp4_quantize(icq.rotate_activations(F.silu(gate) * up, ROT))
    return h + icq.mxfp4_linear(inner, w[NAMES[2]])


def main(argv=None) -> dict[str, float]:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--hidden", type=int, default=1024)
    ap.add_argument("--inner", type=int, default=2816)
    ap.add_argument("--rows", type=int, default=300)
    a = ap.parse_args(argv)
    g = torch.Generator().manual_seed(0)
    state = {n: (torch.randn(a.inner if "down" not in n else a.hidden, a.hidden if "down" not in n else a.inner,
                             generator=g) * 0.02).to(torch.bfloat16) for n in NAMES}
    x, r = (torch.randn(a.rows, a.hidden, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    gain = (1 + 0.1 * torch.randn(a.hidden, generator=g)).to(torch.bfloat16).cuda()
    h = x.double() + r.double()
    n = h / torch.sqrt(h.square().mean(1, keepdim=True) + 1e-6) * gain.double()
    W = [state[k].cuda().double() for k in NAMES]
    branch = (F.silu(n @ W[0].T) * (n @ W[1].T)) @ W[2].T
    errors = {}
    with tempfile.TemporaryDirectory() as folder:
        ways = {"int8": (run_integer, convert(state, 8, folder)), "int4": (run_integer, convert(state, 4, folder)),
                "mxfp4": (run_mxfp4, {k: icq.mxfp4_quantize(icq.rotate_weights(state[k].cuda().float(), ROT))
                                      for k in NAMES})}
    for name, (run, w) in ways.items():
        for label, rows in (("prompt", slice(None)), ("token", slice(0, 1))):
            y = run(x[rows], r[rows], gain, w).double() - h[rows]          # what the block adds
            errors[f"{name} {label}"] = ((y - branch[rows]).norm() / branch[rows].norm()).item()
            print(f"{name:6s} {label:6s} relative error of the block {errors[f'{name} {label}']:.4f}")
    return errors


if __name__ == "__main__":
    main()
