"""Adapters' workspace and what they keep: no GPU."""

from __future__ import annotations

import os

import pytest
import torch

import int_crush_converter_amd as icq
from int_crush_converter_amd import _native as nat
from int_crush_converter_amd import adapters, linear


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(nat.LIB_PATH):
        from int_crush_converter_amd import build
        build.build()
    nat.load(require_gpu=False)
    return nat._lib


def test_the_workspace_is_the_librarys(L):
    for rows in (1, 15, 64, 65, 100, 8192, 1048560):
        for rank in (1, 16, 32, 33, 100, 128):
            assert 4 * linear._adapted_workspace(rows, rank) == L.ic_adapted_linear_workspace_bytes(rows, rank)


@pytest.mark.parametrize("given", [torch.tensor([0.5, 2.0, 3.0]), torch.tensor(2.0), torch.tensor([[2.0]]), torch.tensor([1, 2, 3]), 1.5])
def test_the_scaling_is_a_copy(L, monkeypatch, given):
    """However it was given; host tensors stand for the GPU's."""
    monkeypatch.setattr(nat, "lib", lambda: L)
    monkeypatch.setattr(nat, "on_gpu", lambda name, t: t)
    monkeypatch.setattr(nat, "stream_for", lambda *t: 0)
    monkeypatch.setattr(adapters, "call", lambda name, *args: None)
    given = given.clone() if isinstance(given, torch.Tensor) else given
    for n in (3, 1):
        if isinstance(given, torch.Tensor) and given.numel() not in (1, n):
            continue
        ad = icq.LowRankAdapters(torch.zeros(n, 4, 64, dtype=torch.bfloat16), torch.zeros(n, 16, 4, dtype=torch.bfloat16), given)
        want = torch.as_tensor(given).float().reshape(-1).expand(n).clone()
        assert ad.scaling.dtype == torch.float32 and ad.scaling.is_contiguous() and torch.equal(ad.scaling, want)
        if isinstance(given, torch.Tensor):
            given += 7
            assert torch.equal(ad.scaling, want)
            given -= 7
