"""Low-rank adapters of many requests beside one quantised weight:

    y[m] = quantized_linear(x, weight, bias)[m] + scaling[a] B_a (A_a x[m]),   a = the adapter of row m

x being what the 8-bit activations stand for (``q * s``).  The adapters of a
layer are laid out once; ``quantized_linear(adapters=, groups=)`` runs them."""

from __future__ import annotations

import torch

from . import _native as nat
from .activations import MAX_FEATURES, call
from .groups import MAX_GROUPS

MAX_RANK = 128


class LowRankAdapters:
    """The adapters of one layer: a [count, rank, in_features] and b [count, out_features, rank], both bfloat16 or both
    float16, and their scaling (a number, or [count]); copies are kept.

    Beside a rotated weight the activations are rotated too: give ``rotate_weights(a, rot_size)`` there, whose rows are
    padded like the activations'.  Adapters of smaller rank are padded with zeros to the largest.  b has to be finite; Inf
    or NaN in a reaches the adapter's own rows."""

    __slots__ = ("down", "up", "scaling", "code", "count", "rank", "in_features", "out_features")

    def __init__(self, a: torch.Tensor, b: torch.Tensor, scaling: float | torch.Tensor = 1.0):
        if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2]:
            raise ValueError(f"expected a [count, rank, in] and b [count, out, rank], got {tuple(a.shape)} and {tuple(b.shape)}")
        if a.dtype != b.dtype or a.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"adapters are bfloat16 or float16, got {a.dtype} and {b.dtype}")
        n, r, K = a.shape
        N = b.shape[1]
        if not 1 <= n <= MAX_GROUPS or not 1 <= r <= MAX_RANK or not 1 <= K <= MAX_FEATURES or N < 1:
            raise ValueError(f"1 to {MAX_GROUPS} adapters of rank 1 to {MAX_RANK} and in_features up to {MAX_FEATURES}, got {n}, {r}, {K}")
        if not torch.isfinite(b).all():
            raise ValueError("b holds Inf or NaN, which would reach rows of other adapters")
        a, b = nat.on_gpu("a", a).contiguous(), nat.on_gpu("b", b).contiguous()
        if isinstance(scaling, torch.Tensor):
            if scaling.numel() not in (1, n):
                raise ValueError(f"{scaling.numel()} scalings for {n} adapters")
            s = nat.on_gpu("scaling", scaling).float().reshape(-1)
            self.scaling = s.expand(n).clone(memory_format=torch.contiguous_format)
        else:
            self.scaling = torch.full((n,), float(scaling), dtype=torch.float32, device=a.device)
        self.count, self.rank, self.in_features, self.out_features = n, r, K, N
        self.code = nat.dtype_code(a)
        L = nat.lib()
        self.down = nat.workspace(L.ic_adapter_down_bytes(n, r, K), a.device)
        self.up = nat.workspace(L.ic_adapter_up_bytes(n, N, r, self.code), a.device)
        call("ic_adapter_pack", a.data_ptr(), b.data_ptr(), self.code, n, r, N, K, self.down.data_ptr(), self.up.data_ptr(),
             nat.stream_for(a, b))
