"""Microscaled 4-bit floating point (OCP MX: E2M1 elements, one E8M0 scale
for 32 consecutive columns): quantisation and the product of two operands in
that form, on the matrix cores' scaled 4-bit instructions.

A block's scale is ``2^(floor(log2(max|x|)) - 2)``; elements round to the
nearest E2M1 value, ties to even, at most 6.  A block that holds Inf or NaN
has the scale NaN (byte 255)."""

from __future__ import annotations

import math

import torch

from . import _native as nat
from .activations import MAX_FEATURES, as_rows, call
from .linear import MAX_ROWS, _bias, _out_code

BLOCK = 32


def _sizes(rows: int, K: int) -> None:
    if not 1 <= K <= MAX_FEATURES or rows > MAX_ROWS:
        raise ValueError(f"in_features must be in [1, {MAX_FEATURES}] and rows at most {MAX_ROWS}, got {K}, {rows}")


def _nbytes(rows: int, K: int) -> tuple[int, int]:
    """ic_mxfp4_code_bytes and ic_mxfp4_scale_bytes."""
    return -(-rows // 16) * -(-K // 128) * 1024, -(-rows // 16) * -(-K // 512) * 256


class Mxfp4Tensor:
    """A tensor [*lead, in_features] in microscaled 4-bit form, on the GPU, in the tiles that the products read."""

    __slots__ = ("tiles", "scales", "in_features", "lead", "rows")

    def __init__(self, tiles: torch.Tensor, scales: torch.Tensor, in_features: int, lead, rows: int):
        """tiles and scales: the bytes of csrc/lowbit.hpp's layout, one after another; rows: those of ``lead``.
        ``from_packed`` makes them of row-major codes and scales."""
        _sizes(rows, in_features)
        if rows != math.prod(lead):
            raise ValueError(f"{rows} rows for the shape {tuple(lead)}")
        for name, t, n in zip(("tiles", "scales"), (tiles, scales), _nbytes(rows, in_features)):
            if t.dtype != torch.uint8 or tuple(t.shape) != (n,) or not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"{name} must be contiguous uint8 ({n},) at 16-byte alignment, got {t.dtype} "
                                 f"{tuple(t.shape)}")
        self.tiles, self.scales = tiles, scales
        self.in_features, self.lead, self.rows = in_features, tuple(lead), rows

    @classmethod
    def _empty(cls, lead, rows: int, K: int, dev: torch.device) -> "Mxfp4Tensor":
        t = cls.__new__(cls)                 # of tensors made here, as __init__ wants them
        t.tiles, t.scales = (torch.empty(n, dtype=torch.uint8, device=dev) for n in _nbytes(rows, K))
        t.in_features, t.lead, t.rows = K, tuple(lead), rows
        return t

    @classmethod
    def from_packed(cls, codes: torch.Tensor, scales: torch.Tensor, *, in_features: int | None = None) -> "Mxfp4Tensor":
        """From uint8 codes [..., ceil(K/2)] (even column in the low nibble) and E8M0 bytes [..., ceil(K/32)].
        in_features: K, needed where a row ends in half a byte (default: two a byte)."""
        if codes.dim() < 1 or codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise ValueError(f"expected uint8 codes and scales, got {codes.dtype} and {scales.dtype}")
        K = in_features if in_features is not None else 2 * codes.shape[-1]
        _sizes(0, K)
        lead = codes.shape[:-1]
        have, whole = codes.shape[-1], -(-K // BLOCK) * (BLOCK // 2)
        if have not in ((K + 1) // 2, whole) or tuple(scales.shape) != (*lead, -(-K // BLOCK)):
            raise ValueError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not hold {K} columns")
        rows = codes.numel() // have
        _sizes(rows, K)
        c, s = nat.on_gpu("codes", codes), nat.on_gpu("scales", scales)
        t = cls._empty(lead, rows, K, c.device)
        if rows:
            c, s = as_rows(c), as_rows(s)
            call("ic_mxfp4_relayout", c.data_ptr(), c.stride(0) if rows > 1 else have, s.data_ptr(),
                 s.stride(0) if rows > 1 else s.shape[1], rows, K, t.tiles.data_ptr(), t.scales.data_ptr(), 1,
                 nat.stream_for(c, s))
        return t

    def to_packed(self) -> tuple[torch.Tensor, torch.Tensor]:
        """(codes [*lead, ceil(K/2)], scales [*lead, ceil(K/32)]), the inverse of ``from_packed``."""
        K, rows, dev = self.in_features, self.rows, self.tiles.device
        stream = nat.stream_for(self.tiles, self.scales)
        c = torch.empty((rows, (K + 1) // 2), dtype=torch.uint8, device=dev)
        s = torch.empty((rows, -(-K // BLOCK)), dtype=torch.uint8, device=dev)
        if rows:
            call("ic_mxfp4_relayout", c.data_ptr(), c.shape[1], s.data_ptr(), s.shape[1], rows, K,
                 self.tiles.data_ptr(), self.scales.data_ptr(), 0, stream)
        return c.reshape(*self.lead, c.shape[1]), s.reshape(*self.lead, s.shape[1])

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values [*lead, in_features] in ``dtype`` (exact in bfloat16 and float32)."""
        K, code = self.in_features, _out_code(dtype)
        stream = nat.stream_for(self.tiles, self.scales)
        out = torch.empty((*self.lead, K), dtype=dtype, device=self.tiles.device)
        call("ic_mxfp4_dequantize", self.tiles.data_ptr(), self.scales.data_ptr(), self.rows, K, out.data_ptr(),
             code, K, stream)
        return out


def mxfp4_quantize(x: torch.Tensor) -> Mxfp4Tensor:
    """x [..., K] (float32 / bfloat16 / float16; weights, or activations) in microscaled 4-bit form.  Weights and
    activations that are to be rotated are rotated before (``rotate_weights``, ``rotate_activations``)."""
    if x.dim() < 1:
        raise ValueError("expected [..., K]")
    K = x.shape[-1]
    rows = x.numel() // K if K else 0
    _sizes(rows, K)
    xg = nat.on_gpu("x", x)
    code = nat.dtype_code(xg)
    t = Mxfp4Tensor._empty(x.shape[:-1], rows, K, xg.device)
    if rows:
        xr = as_rows(xg)
        call("ic_mxfp4_quantize", xr.data_ptr(), code, rows, K, xr.stride(0) if rows > 1 else K, t.tiles.data_ptr(),
             t.scales.data_ptr(), nat.stream_for(xr))
    return t


def mxfp4_linear(x: Mxfp4Tensor, weight: Mxfp4Tensor, bias: torch.Tensor | None = None, *,
                 out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """y = x W^T + b [*x.lead, out_features], both operands in microscaled 4-bit form, summed in fp32."""
    if len(weight.lead) != 1 or weight.rows < 1:
        raise ValueError(f"the weight must be 2-D with at least one row, got {(*weight.lead, weight.in_features)}")
    if x.in_features != weight.in_features:
        raise ValueError(f"x has {x.in_features} features, the weight {weight.in_features}")
    N = weight.rows
    code = _out_code(out_dtype)
    b, bcode = _bias(bias, N)
    stream = nat.stream_for(x.tiles, x.scales, weight.tiles, weight.scales)
    out = torch.empty((*x.lead, N), dtype=out_dtype, device=x.tiles.device)
    call("ic_mxfp4_linear", x.tiles.data_ptr(), x.scales.data_ptr(), x.rows, weight.tiles.data_ptr(),
         weight.scales.data_ptr(), None if b is None else b.data_ptr(), bcode, N, x.in_features, out.data_ptr(), code, N,
         stream)
    return out
