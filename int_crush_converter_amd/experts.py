"""Products of rows ordered by expert with the weights that the converter
stored, one for each expert:

    y[i, n] = sa[x(i)] sw_e[n] (sum_k a q_e - zp_e[n] sum_k a) + b_e[n],   e = the expert of place i

x(i) being row i itself, or the token that the pair at place i belongs to
(``gather``: the first product behind a router, whose activations are not
copied).  The sums are exact in 32-bit integers."""

from __future__ import annotations

from collections.abc import Sequence

import torch

from . import _native as nat
from .activations import QuantizedActivations, call
from .groups import MAX_GROUPS, RowGroups
from .linear import QuantizedWeight, _out_code


class ExpertWeight:
    """One layer's weight of every expert, laid out once for ``expert_linear``: copies of ``QuantizedWeight``s of one
    size, one number of bits and one kind of scales, with zero-points or all without."""

    __slots__ = ("tiles", "scales", "scale_kind", "zero_points", "bits", "in_features", "out_features", "experts")

    def __init__(self, layers: Sequence[QuantizedWeight]):
        layers = list(layers)
        if not 1 <= len(layers) <= MAX_GROUPS:
            raise ValueError(f"1 to {MAX_GROUPS} experts, got {len(layers)}")
        form = lambda w: (w.bits, w.in_features, w.out_features, w.scale_kind, w.zero_points is None)      # noqa: E731
        for i, w in enumerate(layers):
            if form(w) != form(layers[0]):
                raise ValueError(f"expert {i} differs from the first (bits, in_features, out_features, scale kind, symmetric): "
                                 f"{form(w)} and {form(layers[0])}")
            nat.stream_for(w.tiles, w.scales, w.zero_points)
        first = layers[0]
        self.bits, self.in_features, self.out_features = first.bits, first.in_features, first.out_features
        self.scale_kind, self.experts = first.scale_kind, len(layers)
        self.tiles = torch.cat([w.tiles for w in layers])
        self.scales = torch.cat([w.scales for w in layers])
        self.zero_points = None if first.zero_points is None else torch.cat([w.zero_points for w in layers])


def expert_linear(x: QuantizedActivations, weight: ExpertWeight, groups: RowGroups, bias: torch.Tensor | None = None, *,
                  gather: bool, out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """y [rows * per_row, out_features] in ``out_dtype``, in the order of ``groups``.

    gather: x has the groups' rows (tokens), each used for all its choices; else x is in the order already, one row a
    place.  bias: [experts, out_features].  out: written instead of a new tensor (its dtype counts).  Places behind the
    last group's (pairs of no expert) are not written.  Rows of x whose scale is NaN give rows of NaN."""
    w, z, pairs = weight, weight.zero_points, groups.rows * groups.per_row
    if x.in_features != w.in_features:
        raise ValueError(f"activations have {x.in_features} features, the weight {w.in_features}")
    if groups.groups != w.experts:
        raise ValueError(f"rows are grouped among {groups.groups}, the weight has {w.experts} experts")
    data, N = x.data, w.out_features
    have = data.shape[0]
    if have != (groups.rows if gather else pairs):
        raise ValueError(f"{have} rows of activations, expected {groups.rows if gather else pairs}")
    b, bcode = None, 0
    if bias is not None:
        if bias.shape != (w.experts, N):
            raise ValueError(f"bias has shape {tuple(bias.shape)}, expected ({w.experts}, {N})")
        b = nat.on_gpu("bias", bias).contiguous()
        bcode = nat.dtype_code(b)
    if out is None:
        code = _out_code(out_dtype)
        stream = nat.stream_for(data, x.meta, w.tiles, w.scales, z, groups.data)
        out = torch.empty((pairs, N), dtype=out_dtype, device=data.device)
    else:
        if tuple(out.shape) != (pairs, N) or (N > 1 and out.stride(1) != 1) or (pairs > 1 and out.stride(0) < N):
            raise ValueError(f"out must be ({pairs}, {N}) with contiguous rows, got {tuple(out.shape)} with strides {out.stride()}")
        code = _out_code(out.dtype)
        stream = nat.stream_for(data, x.meta, w.tiles, w.scales, z, groups.data, out)
    m = x.meta.data_ptr()
    _, offsets, order, _ = groups.pointers()
    call("ic_expert_linear", data.data_ptr(), data.shape[1], m, m + 4 * have, have, offsets, order,
         groups.per_row if gather else 0, w.experts, pairs, w.tiles.data_ptr(), w.bits, w.scales.data_ptr(), w.scale_kind,
         None if z is None else z.data_ptr(), None if b is None else b.data_ptr(), bcode, N, w.in_features, out.data_ptr(),
         code, out.stride(0) if pairs > 1 else N, stream)
    return out
