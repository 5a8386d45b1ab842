"""The example runs, and each format's error is of its step's size: 8 bits
leave about a hundredth, 4 bits about a tenth a product (three products, two
of them multiplied with each other)."""

from __future__ import annotations

import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu


def test_quantized_mlp_example(gpu_dev, capsys):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "run_quantized_mlp.py")
    spec = importlib.util.spec_from_file_location("run_quantized_mlp", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    e = mod.main(["--hidden", "512", "--inner", "1280", "--rows", "70"])
    assert set(e) == {f"{a} {b}" for a in ("int8", "int4", "mxfp4") for b in ("prompt", "token")}
    assert all(v < 0.06 for k, v in e.items() if k.startswith("int8")), e
    assert all(v < 0.5 for v in e.values()), e
    assert "relative error" in capsys.readouterr().out
