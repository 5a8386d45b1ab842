"""Size queries and host-side refusals of the operators' entry points: no GPU."""

from __future__ import annotations

import ctypes
import os

import pytest

from int_crush_converter_amd import _native as nat


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(nat.LIB_PATH):
        from int_crush_converter_amd import build
        build.build()
    nat.load(require_gpu=False)
    return nat._lib


def test_sizes(L):
    assert [L.ic_activation_pitch(n) for n in (1, 128, 129, 12288)] == [128, 128, 256, 12288]
    assert L.ic_linear_weight_bytes(1, 1, 8) == 2048 and L.ic_linear_weight_bytes(17, 129, 4) == 2 * 2 * 1024
    assert L.ic_linear_weight_bytes(16, 16, 5) == 0
    assert L.ic_mxfp4_code_bytes(17, 129) == 2 * 2 * 1024 and L.ic_mxfp4_scale_bytes(17, 513) == 2 * 2 * 256
    assert L.ic_mxfp4_code_bytes(1048560, 65536) == 65535 * 512 * 1024       # past 32 bits


def test_refusals_on_the_host(L):
    one = ctypes.c_void_p(16)          # an address that no refused call touches
    rows = lambda **k: L.ic_quantize_rows(one, k.get("dtype", 0), k.get("rows", 4), k.get("cols", 64), k.get("ld", 64),
                                          None, 0, None, 0, 1e-6, k.get("rot", 1), one, k.get("ldq", 128), one, one,
                                          k.get("ro"), 0, None)                                      # noqa: E731
    assert rows(dtype=3) == -1 and rows(cols=0) == -1 and rows(ld=63) == -1 and rows(ldq=64) == -1
    assert rows(rot=32) == -1 and b"rot must be" in L.ic_last_error()
    assert rows(ro=one) == -1 and b"go together" in L.ic_last_error()
    assert rows(cols=65537, ld=65537, ldq=65664) == -3
    assert rows(rows=0) == 0
    lin = lambda **k: L.ic_quantized_linear(one, k.get("lda", 128), one, None, k.get("M", 4), one, k.get("bits", 4), one,
                                            0, k.get("zp"), None, 0, k.get("N", 8), k.get("K", 64), one,
                                            k.get("out", 1), k.get("ldo", 8), None)                  # noqa: E731
    assert lin(bits=3) == -1 and lin(out=5) == -1 and lin(lda=64) == -1 and lin(lda=136) == -1 and lin(ldo=7) == -1
    assert lin(zp=one) == -1 and b"null" in L.ic_last_error()                # zero-points need the sums
    assert lin(K=65537, lda=65664) == -3 and lin(lda=(1 << 20) + 128) == -3 and lin(M=0) == 0
    assert L.ic_mxfp4_linear(one, one, 4, one, one, None, 0, 8, 64, one, 1, 7, None) == -1
    assert L.ic_mxfp4_quantize(one, 0, 1 << 21, 64, 64, one, one, None) == -3
    assert L.ic_mxfp4_relayout(one, 15, one, 1, 4, 32, one, one, 1, None) == -1
