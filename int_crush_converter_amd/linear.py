"""Products with the weights that the converter stores: ``y = x W^T + b`` for
8-bit activations (``activations.py``) and INT8 or packed INT4 weights with a
scale, and where asymmetric a zero-point, a row:

    y[m, n] = sa[m] sw[n] (sum_k a q - zp[n] sum_k a) + b[n]

The sums are exact in 32-bit integers (int8 matrix instructions)."""

from __future__ import annotations

import torch

from . import _native as nat
from . import packing
from .activations import MAX_FEATURES, QuantizedActivations, as_rows, call

MAX_ROWS = 1048560


_DTYPES = {torch.float32: nat.DT_F32, torch.bfloat16: nat.DT_BF16, torch.float16: nat.DT_F16}


def _out_code(out_dtype: torch.dtype) -> int:
    code = _DTYPES.get(out_dtype)
    if code is None:
        raise TypeError(f"unsupported dtype {out_dtype}")
    return code


def _bias(bias: torch.Tensor | None, N: int):
    if bias is None:
        return None, 0
    if bias.shape != (N,):
        raise ValueError(f"bias has shape {tuple(bias.shape)}, expected ({N},)")
    b = nat.on_gpu("bias", bias).contiguous()
    return b, nat.dtype_code(b)


def _unpermuted(rows: torch.Tensor, permutation: torch.Tensor, bits: int, K: int) -> torch.Tensor:
    """Stored rows with their columns where they were before the converter permuted them: column j of the first
    len(permutation) goes to permutation[j]."""
    if permutation.dim() != 1 or permutation.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"expected a permutation of column numbers, got {permutation.dtype} {tuple(permutation.shape)}")
    p, n = nat.on_gpu("permutation", permutation).long(), permutation.numel()
    if n > K or not torch.equal(p.sort().values, torch.arange(n, device=p.device)):
        raise ValueError(f"not a permutation of the first {n} of {K} columns")
    codes = packing.unpack_int4(rows, K) if bits == 4 else rows
    out = codes.clone()
    out[:, p] = codes[:, :n]
    return packing.pack_int4(out) if bits == 4 else out


class QuantizedWeight:
    """A stored weight laid out once for ``quantized_linear``.

    stored: int8 [N, K] (INT8) or uint8 [N, ceil(K/2)] (INT4, low nibble first); scales: fp16 or fp32 [N] or [N, 1];
    zero_points: int8 of the same shape, or None; permutation: int32 or int64, up to K column numbers, or None -
    ``<name>``, ``<name>_scale``, ``<name>_zp`` and ``<name>_perm`` of the converter's output.  A permuted layer's
    columns are put back in order here, so that its activations are those of any other layer; without its
    permutation its products are wrong.  in_features: K, needed where an INT4 row ends in half a byte."""

    __slots__ = ("tiles", "scales", "scale_kind", "zero_points", "bits", "in_features", "out_features")

    def __init__(self, stored: torch.Tensor, scales: torch.Tensor, zero_points: torch.Tensor | None = None, *,
                 permutation: torch.Tensor | None = None, in_features: int | None = None):
        if stored.dim() != 2 or stored.dtype not in (torch.int8, torch.uint8):
            raise ValueError(f"expected int8 [N, K] or packed uint8 [N, ceil(K/2)], got {stored.dtype} {tuple(stored.shape)}")
        N, width = stored.shape
        bits = 8 if stored.dtype == torch.int8 else 4
        K = in_features if in_features is not None else width * (1 if bits == 8 else 2)
        if (K if bits == 8 else (K + 1) // 2) != width:
            raise ValueError(f"in_features {K} does not fit rows of {width} bytes ({bits} bits)")
        if not 1 <= K <= MAX_FEATURES or not 1 <= N <= MAX_ROWS:
            raise ValueError(f"in_features must be in [1, {MAX_FEATURES}] and out_features in [1, {MAX_ROWS}], got {K}, {N}")
        if scales.numel() != N or (zero_points is not None and zero_points.numel() != N):
            raise ValueError(f"{N} rows need {N} scales and zero-points: one a row")
        s = nat.on_gpu("scales", scales).reshape(-1)
        self.scales = (s if s.dtype in (torch.float16, torch.float32) else s.float()).contiguous()
        self.scale_kind = 0 if self.scales.dtype == torch.float16 else 1
        if zero_points is not None and zero_points.dtype != torch.int8:
            raise ValueError(f"zero_points must be int8, got {zero_points.dtype}")
        self.zero_points = None if zero_points is None else nat.on_gpu("zero_points", zero_points).reshape(-1).contiguous()
        self.bits, self.in_features, self.out_features = bits, K, N
        rows = as_rows(nat.on_gpu("stored", stored))
        if permutation is not None:
            rows = _unpermuted(rows, permutation, bits, K)
        self.tiles = nat.workspace(nat.lib().ic_linear_weight_bytes(N, K, bits), rows.device)
        call("ic_linear_pack_weight", rows.data_ptr(), bits, N, K, rows.stride(0) if N > 1 else width,
             self.tiles.data_ptr(), nat.stream_for(rows))


def quantized_linear(x: QuantizedActivations, weight: QuantizedWeight, bias: torch.Tensor | None = None, *,
                     out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """y [*lead, out_features] in ``out_dtype``.  Rows of x whose scale is NaN give rows of NaN."""
    if x.in_features != weight.in_features:
        raise ValueError(f"activations have {x.in_features} features, the weight {weight.in_features}")
    data, N, w, z = x.data, weight.out_features, weight, weight.zero_points
    code = _out_code(out_dtype)
    b, bcode = _bias(bias, N)
    stream = nat.stream_for(data, x.meta, w.tiles, w.scales, z)
    out = torch.empty((*x.lead, N), dtype=out_dtype, device=data.device)
    rows, m = data.shape[0], x.meta.data_ptr()
    call("ic_quantized_linear", data.data_ptr(), data.shape[1], m, m + 4 * rows, rows, w.tiles.data_ptr(), w.bits,
         w.scales.data_ptr(), w.scale_kind, None if z is None else z.data_ptr(), None if b is None else b.data_ptr(),
         bcode, N, w.in_features, out.data_ptr(), code, N, stream)
    return out
