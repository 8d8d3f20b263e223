"""What the operators on 8-bit values with block scales and the orthogonalised updates refuse when they are created, before
they touch a device, and null handles at the C entries."""
import pytest

import ccglib_amd as cc
from ccglib_amd import _capi

VT, SG, ST = cc.ValueType, cc.ScaleGroup, cc.ScaleType


def test_pitch():
    assert [cc.scaled_pitch(n) for n in (0, 1, 16, 17, 128)] == [0, 16, 16, 32, 128]


@pytest.mark.parametrize("change,message", [
    (dict(input_type=VT.float8e4m3), "input is float32"), (dict(input_type=VT.int1), "input is float32"),
    (dict(output_type=VT.bfloat16), "output is float8e4m3"), (dict(group=2), "out of range"), (dict(scale_type=-1), "out of range"),
    (dict(input_pitch=15), "at a distance"), (dict(M=1 << 31), "size out of range"), (dict(B=1 << 30, M=1 << 20), "size out of range")])
def test_quantize_refuses(change, message):
    args = dict(B=1, M=4, N=16, device=0, stream=0, input_type=VT.float32)
    args.update(change)
    with pytest.raises(RuntimeError, match=message):
        cc.Quantize(**args)


@pytest.mark.parametrize("change,message", [
    (dict(a_type=VT.float16), "operands are float8"), (dict(b_type=VT.int1), "operands are float8"),
    (dict(c_type=VT.float8e5m2), "C is float32"), (dict(c_type=VT.bfloat16, accumulate=True), "added to is float32"),
    (dict(a_group=7), "out of range"), (dict(scale_type=2), "out of range"), (dict(pitch_a=24), "multiple of 16"),
    (dict(pitch_b=16), "multiple of 16"), (dict(pitch_c=7), "at a distance"), (dict(K=(1 << 23) + 1), "size out of range"),
    (dict(M=1 << 30, N=1 << 30), "size out of range")])
def test_scaled_gemm_refuses(change, message):
    args = dict(B=1, M=8, N=8, K=32, device=0, stream=0)
    args.update(change)
    with pytest.raises(RuntimeError, match=message):
        cc.ScaledGEMM(**args)


@pytest.mark.parametrize("change,message", [
    (dict(type=VT.float8e4m3), "input is float32"), (dict(gradient_type=VT.float16), "output is float8e4m3"),
    (dict(scale_type=5), "out of range"), (dict(K=1 << 24), "size out of range")])
def test_scaled_linear_refuses(change, message):
    args = dict(M=8, N=8, K=32, device=0, stream=0)
    args.update(change)
    with pytest.raises(RuntimeError, match=message):
        cc.ScaledLinear(**args)


@pytest.mark.parametrize("change,message", [
    (dict(type=VT.float8e4m3), "matrices are float32"), (dict(steps=0), "1 to 1000 steps"), (dict(epsilon=-1.0), "epsilon"),
    (dict(epsilon=float("nan")), "epsilon"), (dict(input_pitch=7), "at a distance"), (dict(output_pitch=7), "at a distance"),
    (dict(B=65536), "size out of range"), (dict(M=(1 << 20) + 1), "size out of range")])
def test_orthogonalize_refuses(change, message):
    args = dict(B=1, M=8, N=8, device=0, stream=0)
    args.update(change)
    with pytest.raises(RuntimeError, match=message):
        cc.Orthogonalize(**args)


def test_null_handles_are_errors_not_crashes():
    lib = _capi.load()
    assert lib.ccglib_quantize_run(None, None, None, None, None, None) != 0
    assert lib.ccglib_scaled_gemm_run(None, None, None, None, None, None) != 0
    assert lib.ccglib_scaled_gemm_kernel_name(None, None, 0) != 0
    assert lib.ccglib_scaled_linear_set_weights(None, None) != 0
    assert lib.ccglib_scaled_linear_forward(None, None, None) != 0
    assert lib.ccglib_scaled_linear_backward(None, None, None, None, 0) != 0
    assert lib.ccglib_orthogonalize_run(None, None, None) != 0
    assert b"null" in lib.ccglib_last_error()
    assert lib.ccglib_quantize_create(None, 1, 1, 1, 0, None, 6, 3, 0, 0, 0) != 0
    assert lib.ccglib_scaled_gemm_create(None, 1, 1, 1, 1, 0, None, 3, 3, 6, 0, 0, 0, 0, 0, 0, 0) != 0
    assert lib.ccglib_scaled_linear_create(None, 1, 1, 1, 0, None, 6, 3, 0, 1) != 0
    assert lib.ccglib_orthogonalize_create(None, 1, 1, 1, 0, None, 6, 5, 1.0, 1.0, 1.0, 0.0, 0, 0) != 0
    for name in ("quantize", "scaled_gemm", "scaled_linear", "orthogonalize"):
        assert getattr(lib, "ccglib_%s_destroy" % name)(None) == 0
