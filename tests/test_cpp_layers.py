"""Runs the C++ caller of FusedLinear, GroupedLinear, Route and Combine (tests/cpp/layers.cpp)."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
BINARY = os.path.join(HERE, "cpp", "layers")


@pytest.mark.gpu
def test_cpp_layers():
    if not os.path.exists(BINARY):
        subprocess.check_call(["make", "-C", os.path.join(HERE, "cpp"), "layers"])
    r = subprocess.run([BINARY], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "all checks passed" in r.stdout


def test_headers_declare_the_layers():
    inc = os.path.join(os.path.dirname(HERE), "include", "ccglib")
    names = {"pipeline/fused_linear.h": ["class FusedLinear"], "pipeline/grouped_linear.h": ["class GroupedLinear"],
             "route/route.h": ["class Route", "class Combine"]}
    everything = open(os.path.join(inc, "ccglib.hpp")).read()
    for name, declared in names.items():
        text = open(os.path.join(inc, name)).read()
        assert all(d in text for d in declared)
        assert "ccglib/" + name in everything
