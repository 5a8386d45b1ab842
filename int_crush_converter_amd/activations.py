"""8-bit activations for layers that the converter quantised.

``rms_norm_quantize`` and ``quantize_activations`` turn rows of 16- or 32-bit
activations into int8 codes with one fp32 scale a row (``q * s``, ``s`` the
largest magnitude / 127, halves rounded away from zero like the weights'
codes), after the regular-Hadamard rotation that the weights had
(``rotate_weights``): ``W x = (W R^T)(R x)``.  One pass of the HIP library
(``ic_quantize_rows``) adds the residual, normalises, rotates and quantises.
"""

from __future__ import annotations

import math

import torch

from . import _native as nat

ROT_SIZES = (1, 4, 16, 64, 256)
MAX_FEATURES = 65536
_PAD = 128                       # ic_activation_pitch


def as_rows(t: torch.Tensor) -> torch.Tensor:
    """[..., K] as 2-D rows whose columns are contiguous (a copy only where the strides ask for one)."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.stride(1) != 1 and t.shape[1] > 1 or (t.stride(0) < t.shape[1] and t.shape[0] > 1):
        t = t.contiguous()
    return t


_entries: dict[str, object] = {}


def call(name: str, *args) -> None:
    """A library call with the addresses of tensors that ``nat.stream_for`` has checked."""
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = nat.entry(name)
    rc = fn(*args)
    if rc:
        nat.check(rc, name)


class QuantizedActivations:
    """int8 codes of shape ``[*lead, in_features]``, their fp32 scales and the int32 sums of each row's codes.
    On the GPU; rows are stored at a pitch of whole 128 bytes, zeros behind the last column."""

    __slots__ = ("data", "meta", "in_features", "lead")

    def __init__(self, data: torch.Tensor, meta: torch.Tensor, in_features: int, lead):
        """data: int8 [rows, pitch], rows of ``lead`` in order, the pitch in_features padded to 128; meta: fp32 [2, rows],
        the scales and the sums' bits.  ``from_codes`` makes them of codes and scales."""
        rows, pitch = math.prod(lead), -(-in_features // _PAD) * _PAD
        if not 1 <= in_features <= MAX_FEATURES:
            raise ValueError(f"in_features must be in [1, {MAX_FEATURES}], got {in_features}")
        for name, t, dtype, shape in (("data", data, torch.int8, (rows, pitch)), ("meta", meta, torch.float32, (2, rows))):
            if t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"{name} must be contiguous {dtype} {shape} at 16-byte alignment, got {t.dtype} "
                                 f"{tuple(t.shape)} with strides {t.stride()}")
        self.data, self.meta, self.in_features, self.lead = data, meta, in_features, tuple(lead)

    @classmethod
    def _of(cls, data, meta, in_features, lead) -> "QuantizedActivations":
        q = cls.__new__(cls)                 # of tensors made here, as __init__ wants them
        q.data, q.meta, q.in_features, q.lead = data, meta, in_features, tuple(lead)
        return q

    @property
    def scales(self) -> torch.Tensor:
        """fp32 [rows]."""
        return self.meta[0]

    @property
    def sums(self) -> torch.Tensor:
        """int32 [rows]: the sum of each row's codes."""
        return self.meta[1].view(torch.int32)

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scales: torch.Tensor) -> "QuantizedActivations":
        """Codes [..., K] (int8) and scales [...] from elsewhere.  Both are copied: the rows' sums are kept beside them."""
        if codes.dim() < 1 or codes.dtype != torch.int8:
            raise ValueError(f"expected int8 codes [..., K], got {codes.dtype} {tuple(codes.shape)}")
        lead, K = codes.shape[:-1], codes.shape[-1]
        if not 1 <= K <= MAX_FEATURES:
            raise ValueError(f"in_features must be in [1, {MAX_FEATURES}], got {K}")
        codes = as_rows(nat.on_gpu("codes", codes)) if codes.numel() else nat.on_gpu("codes", codes).reshape(-1, K)
        rows = codes.shape[0]
        if scales.numel() != rows:
            raise ValueError(f"{scales.numel()} scales for {rows} rows of codes")
        meta = torch.empty((2, rows), dtype=torch.float32, device=codes.device)
        meta[0] = nat.on_gpu("scales", scales).reshape(-1)
        pitch = -(-K // _PAD) * _PAD
        data = (torch.zeros if pitch > K else torch.empty)((rows, pitch), dtype=torch.int8, device=codes.device)
        data[:, :K] = codes
        call("ic_row_sums_i8", data.data_ptr(), rows, K, data.shape[1], meta.data_ptr() + 4 * rows,
             nat.stream_for(data, meta))
        return cls._of(data, meta, K, lead)

    @property
    def codes(self) -> torch.Tensor:
        """The int8 codes [*lead, in_features] (a view for 2-D activations)."""
        c = self.data[:, : self.in_features]
        return c if len(self.lead) == 1 else c.reshape(*self.lead, self.in_features)

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values ``q * s`` [*lead, in_features], rounded once to ``dtype``."""
        K, data = self.in_features, self.data
        stream = nat.stream_for(data, self.meta)
        out = torch.empty((*self.lead, K), dtype=dtype, device=data.device)
        call("ic_dequantize_rows", data.data_ptr(), data.shape[0], K, data.shape[1], self.meta.data_ptr(),
             out.data_ptr(), nat.dtype_code(out), K, stream)
        return out


def _quantize(x, weight, residual, eps, rot_size):
    if rot_size not in ROT_SIZES and rot_size != 0:
        raise ValueError(f"rot_size must be 0 or one of {ROT_SIZES}, got {rot_size}: rotate_activations serves others")
    if x.dim() < 1:
        raise ValueError("expected activations [..., K]")
    lead, K = x.shape[:-1], x.shape[-1]
    rot = rot_size or 1
    Kp = -(-K // rot) * rot
    if not 1 <= K or Kp > MAX_FEATURES:
        raise ValueError(f"in_features (padded to the rotation) must be in [1, {MAX_FEATURES}], got {K}")
    xg = nat.on_gpu("x", x)
    code = nat.dtype_code(xg)
    dev, rows = xg.device, x.numel() // K
    xr = as_rows(xg) if rows else xg.reshape(0, K)
    rr = out = w = None
    wcode = code
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError(f"residual {tuple(residual.shape)} {residual.dtype} does not match x {tuple(x.shape)} {x.dtype}")
        rg = nat.on_gpu("residual", residual)
        rr = as_rows(rg) if rows else rg.reshape(0, K)
        out = torch.empty(x.shape, dtype=x.dtype, device=dev)
    if weight is not None:
        if weight.shape != (K,):
            raise ValueError(f"the norm's weight has shape {tuple(weight.shape)}, expected ({K},)")
        w = nat.on_gpu("weight", weight)
        if w.dtype != x.dtype:
            if w.dtype not in (torch.float32, torch.bfloat16, torch.float16):
                raise TypeError(f"unsupported dtype {w.dtype}")
            w, wcode = w.float(), nat.DT_F32
        w = w.contiguous()
    pitch = -(-Kp // _PAD) * _PAD
    data = torch.empty((rows, pitch), dtype=torch.int8, device=dev)
    meta = torch.empty((2, rows), dtype=torch.float32, device=dev)
    m = meta.data_ptr()
    call("ic_quantize_rows", xr.data_ptr(), code, rows, K, xr.stride(0) if rows > 1 else K,
         None if rr is None else rr.data_ptr(), 0 if rr is None else rr.stride(0) if rows > 1 else K,
         None if w is None else w.data_ptr(), wcode, eps, rot, data.data_ptr(), pitch, m, m + 4 * rows,
         None if out is None else out.data_ptr(), K, nat.stream_for(xr, rr, w))
    if out is not None and x.device.type != "cuda":
        out = out.to(x.device)
    return QuantizedActivations._of(data, meta, Kp, lead), out


def rms_norm_quantize(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *,
                      eps: float = 1e-6, rot_size: int = 0) -> tuple[QuantizedActivations, torch.Tensor | None]:
    """``h = x + residual``; 8-bit codes of ``rotate(h * rsqrt(mean(h^2) + eps) * weight)``.

    x: [..., K] float32 / bfloat16 / float16; residual: like x or None; weight: [K].  rot_size: 0 (none), 4, 16, 64
    or 256, the size the weights were rotated with; rows are zero-padded to a multiple of it.  Returns the activations
    and ``h`` in x's dtype (None without a residual).  The norm sees the fp32 sum, not its rounding, and holds for any
    finite row.  A row that holds Inf or NaN, or whose rotated values pass a quarter of fp32's range, gets the scale
    NaN and codes 0, and leaves the other rows as they are."""
    if weight is None:
        raise ValueError("rms_norm_quantize needs the norm's weight; quantize_activations is the form without a norm")
    return _quantize(x, weight, residual, float(eps), rot_size)


def quantize_activations(x: torch.Tensor, *, rot_size: int = 0) -> QuantizedActivations:
    """8-bit codes of the (rotated) rows of x [..., K], as rms_norm_quantize without residual and norm."""
    return _quantize(x, None, None, 0.0, rot_size)[0]
