"""Adapters' workspace and what they keep: no GPU."""

from __future__ import annotations

import os

import pytest

from int_crush_converter_amd import _native as nat
from int_crush_converter_amd import linear


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
