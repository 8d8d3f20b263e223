"""Runs the C++ caller of Quantize, ScaledGEMM, ScaledLinear and Orthogonalize (tests/cpp/operators.cpp)."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
BINARY = os.path.join(HERE, "cpp", "operators")


@pytest.mark.gpu
def test_cpp_operators():
    if not os.path.exists(BINARY):
        subprocess.check_call(["make", "-C", os.path.join(HERE, "cpp"), "operators"])
    r = subprocess.run([BINARY], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "all checks passed" in r.stdout


def test_headers_declare_the_operators():
    inc = os.path.join(os.path.dirname(HERE), "include", "ccglib")
    names = {"quantize/quantize.h": "class Quantize", "gemm/scaled_gemm.h": "class ScaledGEMM",
             "pipeline/scaled_linear.h": "class ScaledLinear", "orthogonalize/orthogonalize.h": "class Orthogonalize"}
    everything = open(os.path.join(inc, "ccglib.hpp")).read()
    for name, declared in names.items():
        assert declared in open(os.path.join(inc, name)).read()
        assert "ccglib/" + name in everything
