"""Rows of activations ordered by the group they belong to: the experts that a
router chose for each token, or the adapter of each row's request.

``route_tokens`` chooses and orders, ``group_rows`` orders given numbers;
``expert_linear`` and ``quantized_linear(adapters=)`` read the order, and
``combine_experts`` brings the experts' rows back to their tokens:

    w[t, j] = exp(x[t, e_j] - max x) / sum,   y[t] = r[t] + sum_j w[t, j] z[position[t, j]]

Everything stays on the GPU: the number of rows that a group got is not read
back, and the same calls can be replayed from a graph with other choices."""

from __future__ import annotations

import torch

from . import _native as nat
from .activations import as_rows, call

MAX_GROUPS, MAX_CHOICES, MAX_PAIRS = 1024, 64, 1048560


def _gpu(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_cuda else nat.to_gpu(t)          # (which GPU: nat.stream_for asks, of all operands at once)


class RowGroups:
    """The (row, choice) pairs of a batch ordered by group, in int32 on the GPU; pair p is choice ``p % per_row`` of row
    ``p // per_row``.  Made by ``group_rows`` and ``route_tokens``."""

    __slots__ = ("data", "scratch", "rows", "per_row", "groups")

    def __init__(self, *args, **kwargs):
        raise TypeError("RowGroups are made by group_rows and route_tokens")

    @classmethod
    def _empty(cls, rows: int, per_row: int, groups: int, dev: torch.device) -> "RowGroups":
        if not 1 <= groups <= MAX_GROUPS or not 1 <= per_row <= MAX_CHOICES or rows * per_row > MAX_PAIRS:
            raise ValueError(f"at most {MAX_GROUPS} groups, {MAX_CHOICES} choices a row and {MAX_PAIRS} pairs, got {groups}, "
                             f"{per_row} and {rows} rows")
        # one allocation: workspace (ic_group_workspace_bytes: 16-bit counts of at most 256 units of at least 16 rows), ids,
        # order, position, offsets
        g = cls.__new__(cls)
        g.scratch = min(256, (rows + 15) // 16) * ((groups + 7) // 8) * 4
        g.data = torch.empty(g.scratch + 3 * rows * per_row + groups + 1, dtype=torch.int32, device=dev)
        g.rows, g.per_row, g.groups = rows, per_row, groups
        return g

    def pointers(self) -> tuple[int, int, int, int]:
        """Addresses of ids, offsets, order and position."""
        at, n = self.data.data_ptr() + 4 * self.scratch, 4 * self.rows * self.per_row
        return at, at + 3 * n, at + n, at + 2 * n

    def _part(self, i: int, flat: bool) -> torch.Tensor:
        n = self.rows * self.per_row
        shape, strides = ((n,), (1,)) if flat else ((self.rows, self.per_row), (self.per_row, 1))
        return self.data.as_strided(shape, strides, self.scratch + i * n)

    @property
    def ids(self) -> torch.Tensor:
        """int32 [rows, per_row]: each pair's group, -1 for none."""
        return self._part(0, False)

    @property
    def offsets(self) -> torch.Tensor:
        """int32 [groups + 1]: group g has the places offsets[g] to offsets[g + 1] - 1 of the order."""
        return self.data[self.scratch + 3 * self.rows * self.per_row:]

    @property
    def order(self) -> torch.Tensor:
        """int32 [rows * per_row]: the pair at each place, -1 behind the last group's."""
        return self._part(1, True)

    @property
    def position(self) -> torch.Tensor:
        """int32 [rows, per_row]: each pair's place, -1 for none."""
        return self._part(2, False)


def group_rows(ids: torch.Tensor, groups: int) -> RowGroups:
    """The order of ids [rows] or [rows, per_row] (int32 or int64) by group; equal ones keep their order.  Numbers outside
    [0, groups) mean none: such pairs are in no group."""
    if ids.dim() not in (1, 2) or ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"expected int32 or int64 ids [rows] or [rows, per_row], got {ids.dtype} {tuple(ids.shape)}")
    given = _gpu(ids).contiguous()
    g = RowGroups._empty(ids.shape[0], ids.shape[1] if ids.dim() == 2 else 1, groups, given.device)
    to, offsets, order, position = g.pointers()
    call("ic_group_rows", given.data_ptr(), int(given.dtype == torch.int64), g.rows, g.per_row, groups, to, offsets, order,
         position, g.data.data_ptr(), nat.stream_for(given))
    return g


def route_tokens(logits: torch.Tensor, top: int, *, renormalize: bool = True) -> tuple[RowGroups, torch.Tensor]:
    """The ``top`` largest of each row of logits [tokens, experts] (float32 / bfloat16 / float16) in order of experts, and
    their fp32 weights [tokens, top].

    Choices are the largest first, of equals the lowest expert.  An expert whose logit is -inf is never chosen: where
    fewer than ``top`` are left, the choice is none (id and position -1, weight 0), and a token of which none is left is in no
    group.  Weights are softmax over all experts, divided by their sum over the chosen if ``renormalize``.  NaN counts
    as the largest; a token with NaN or +inf has weights NaN."""
    if logits.dim() != 2:
        raise ValueError(f"expected logits [tokens, experts], got {tuple(logits.shape)}")
    tokens, experts = logits.shape
    if not 1 <= top <= experts:
        raise ValueError(f"top must be in [1, {experts}] (the experts), got {top}")
    x = _gpu(logits)
    code = nat.dtype_code(x)
    g = RowGroups._empty(tokens, top, experts, x.device)
    x = as_rows(x) if tokens else x
    weights = torch.empty((tokens, top), dtype=torch.float32, device=x.device)
    ids, offsets, order, position = g.pointers()
    call("ic_route_tokens", x.data_ptr(), code, tokens, experts, x.stride(0) if tokens > 1 else experts, top,
         int(renormalize), ids, weights.data_ptr(), offsets, order, position, g.data.data_ptr(), nat.stream_for(x))
    return g, weights if logits.is_cuda else weights.to(logits.device)


def combine_experts(y: torch.Tensor, groups: RowGroups, weights: torch.Tensor, residual: torch.Tensor | None = None
                    ) -> torch.Tensor:
    """[tokens, features] in y's dtype: the weighted sum of each token's rows of y [tokens * top, features], which are in
    the order of ``groups``, and ``residual`` [tokens, features] (or None), rounded once.  weights: [tokens, top], as
    ``route_tokens`` gives them.  Choices that are none add nothing, whatever their weight."""
    pairs = groups.rows * groups.per_row
    if y.dim() != 2 or y.shape[0] != pairs or y.shape[1] < 1:
        raise ValueError(f"expected y [{pairs}, features], got {tuple(y.shape)}")
    cols = y.shape[1]
    if tuple(weights.shape) != (groups.rows, groups.per_row) or not weights.is_floating_point():
        raise ValueError(f"expected weights ({groups.rows}, {groups.per_row}), got {weights.dtype} {tuple(weights.shape)}")
    yr = _gpu(y)
    code = nat.dtype_code(yr)
    w = _gpu(weights)
    if w.dtype != torch.float32 or not w.is_contiguous():
        w = w.float().contiguous()
    r = None
    if residual is not None:
        if tuple(residual.shape) != (groups.rows, cols) or residual.dtype != y.dtype:
            raise ValueError(f"residual {tuple(residual.shape)} {residual.dtype} does not match ({groups.rows}, {cols}) {y.dtype}")
        r = _gpu(residual)
    stream = nat.stream_for(yr, w, r, groups.data)
    if groups.rows:
        yr, r = as_rows(yr), None if r is None else as_rows(r)
    out = torch.empty((groups.rows, cols), dtype=y.dtype, device=yr.device)
    call("ic_combine_rows", yr.data_ptr(), code, groups.rows, groups.per_row, cols, yr.stride(0) if pairs > 1 else cols,
         groups.pointers()[3], w.data_ptr(), None if r is None else r.data_ptr(),
         0 if r is None else r.stride(0) if groups.rows > 1 else cols, out.data_ptr(), cols, stream)
    return out if y.is_cuda else out.to(y.device)
