"""The memory of a ScaledLinear: its products share counters and partial sums, and no product's partial sums may lie on
counters, which have to be zero whenever a product starts, or on a copy of x, W or dy. What the kernels are handed is
recorded without a GPU (tests/cpp/scaled_linear_layout.hip)."""
import ctypes
import math
import os
import random
import subprocess

import pytest

import ccglib_amd as cc

HERE = os.path.dirname(os.path.abspath(__file__))
VT, ST = cc.ValueType, cc.ScaleType


@pytest.fixture(scope="module")
def layout():
    subprocess.check_call(["make", "-C", os.path.join(HERE, "cpp"), "libscaled_linear_layout.so"],
                          stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
    lib = ctypes.CDLL(os.path.join(HERE, "cpp", "libscaled_linear_layout.so"))
    sz, pointer = ctypes.c_size_t, ctypes.POINTER(ctypes.c_size_t)
    lib.scaled_linear_layout.argtypes = [sz, sz, sz, ctypes.c_int, ctypes.c_int, ctypes.c_int, sz, pointer, pointer]

    def call(M, N, K, t, tg=VT.float8e5m2, st=ST.float32, option=0):
        ranges, sizes = (sz * 36)(), (sz * 2)()
        lib.scaled_linear_layout(M, N, K, int(t), int(tg), int(st), option, ranges, sizes)
        pairs = list(zip(ranges[::2], ranges[1::2]))
        return pairs[0:6:2], pairs[1:6:2], pairs[6:], sizes[0], sizes[1]
    return call


def apart(a, b):
    return a[0] == a[1] or b[0] == b[1] or a[1] <= b[0] or b[1] <= a[0]


def check(layout, *args, **more):
    """Returns how many counters each product has."""
    counters, sums, copies, size, cleared = layout(*args, **more)
    for r in counters:
        assert r[0] == r[1] or r[1] <= cleared, (args, more)
    for s in sums:
        assert all(apart(s, r) for r in counters + copies), (args, more)
    for i, c in enumerate(copies):
        assert all(apart(c, r) for r in counters + copies[:i]), (args, more)
    assert all(r[1] <= size for r in counters + sums + copies if r[0] < r[1]), (args, more)
    return [(r[1] - r[0]) // 4 for r in counters]


@pytest.mark.parametrize("M,N,K,t,st", [
    (32, 2560, 5120, VT.float32, ST.float32), (32, 5120, 2560, VT.float32, ST.float32), (16, 4096, 8192, VT.float32, ST.float32),
    (2649, 127, 5376, VT.bfloat16, ST.float32), (180, 4441, 6379, VT.float32, ST.e8m0)])
def test_products_with_unlike_counters(layout, M, N, K, t, st):
    """Layers two of whose products cut K into parts, one with more than the other's counters and 64 besides."""
    n = [c for c in check(layout, M, N, K, t, VT.float8e5m2, st) if c]
    assert len(n) >= 2 and max(n) > 64


def test_any_layer(layout):
    rng = random.Random(1)
    unlike = 0
    for _ in range(4000):
        M, N, K = (int(round(math.exp(rng.uniform(math.log(1), math.log(8192))))) for _ in range(3))
        option = rng.choice([0, 0, 0, 1 + rng.randrange(6) + 256 * rng.randrange(20)])
        n = check(layout, M, N, K, rng.choice([VT.float32, VT.float16, VT.bfloat16]), rng.choice([VT.float8e4m3, VT.float8e5m2]),
                  rng.choice(list(ST)), option=option)
        unlike += len({-(-c // 64) for c in n if c}) > 1
    assert unlike > 100       # (the layers that this is about)
