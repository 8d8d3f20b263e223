"""What the 16-bit linear layers, those grouped by expert, and the routing operators refuse when they are created, before they
touch a device, and null handles at the C entries."""
import pytest

import ccglib_amd as cc
from ccglib_amd import _capi

VT = cc.ValueType
LAYER = [
    (dict(type=VT.float32), "values are float16"), (dict(type=VT.float8e4m3), "values are float16"),
    (dict(gradient_type=VT.float16), "gradients of weights"), (dict(gradient_type=VT.int1), "gradients of weights"),
    (dict(activation=4), "out of range"), (dict(activation=-1), "out of range"), (dict(x_pitch=31), "at distances"),
    (dict(w_pitch=31), "at distances"), (dict(y_pitch=7), "at distances"), (dict(y_pitch=(1 << 22) + 1), "at distances"),
    (dict(K=(1 << 22) + 1), "size out of range"), (dict(N=(1 << 22) + 1), "size out of range"), (dict(M=1 << 31), "size out of range"),
    (dict(M=(1 << 31) - 1, N=1 << 22, K=1), "more blocks than a launch"), (dict(M=1 << 23, K=1), "more blocks than a launch")]


@pytest.mark.parametrize("change,message", LAYER)
def test_fused_linear_refuses(change, message):
    with pytest.raises(RuntimeError, match=message):
        cc.FusedLinear(**(dict(M=8, N=8, K=32, device=0, stream=0) | change))


@pytest.mark.parametrize("change,message", LAYER + [(dict(E=0), "experts"), (dict(E=1025), "experts")])
def test_grouped_linear_refuses(change, message):
    with pytest.raises(RuntimeError, match=message):
        cc.GroupedLinear(**(dict(E=4, M=8, N=8, K=32, device=0, stream=0) | change))


@pytest.mark.parametrize("change,message", [
    (dict(type=VT.float8e5m2), "logits are float32"), (dict(E=0), "experts"), (dict(E=1025), "experts"), (dict(k=0), "chosen"),
    (dict(k=17), "chosen"), (dict(E=3, k=4), "chosen"), (dict(T=1 << 24), "size out of range")])
def test_route_refuses(change, message):
    with pytest.raises(RuntimeError, match=message):
        cc.Route(**(dict(T=8, E=32, k=2, device=0, stream=0) | change))


@pytest.mark.parametrize("change,message", [
    (dict(type=VT.float32), "values are float16"), (dict(k=0), "rows a token"), (dict(k=17), "rows a token"),
    (dict(T=1 << 24), "size out of range"), (dict(rows=1 << 31), "size out of range"), (dict(N=(1 << 22) + 1), "size out of range"),
    (dict(y_pitch=7), "at distances"), (dict(out_pitch=7), "at distances")])
def test_combine_refuses(change, message):
    with pytest.raises(RuntimeError, match=message):
        cc.Combine(**(dict(T=8, k=2, N=8, device=0, stream=0) | change))


def test_null_handles_are_errors_not_crashes():
    lib = _capi.load()
    calls = {"fused_linear_forward": 6, "grouped_linear_forward": 7, "route_run": 5, "route_backward": 5, "combine_run": 4,
             "combine_spread": 4, "combine_backward": 6}
    for name, pointers in calls.items():
        assert getattr(lib, "ccglib_" + name)(None, *[None] * pointers) != 0
        assert b"null handle" in lib.ccglib_last_error()
    assert lib.ccglib_fused_linear_backward(None, *[None] * 7, 0) != 0
    assert lib.ccglib_grouped_linear_backward(None, *[None] * 8, 0) != 0
    assert lib.ccglib_fused_linear_kernel_name(None, 0, None, 0) != 0
    assert lib.ccglib_grouped_linear_kernel_name(None, 0, None, 0) != 0
    assert lib.ccglib_fused_linear_create(None, 1, 1, 1, 0, None, 2, 0, 2, 1, 0, 0, 0) != 0
    assert lib.ccglib_grouped_linear_create(None, 1, 1, 1, 1, 0, None, 2, 0, 2, 1, 0, 0, 0) != 0
    assert lib.ccglib_route_create(None, 1, 1, 1, 0, None, 6, 1) != 0
    assert lib.ccglib_combine_create(None, 1, 1, 1, 0, None, 2, 0, 0, 0) != 0
    for name in ("fused_linear", "grouped_linear", "route", "combine"):
        assert getattr(lib, "ccglib_%s_destroy" % name)(None) == 0


@pytest.mark.parametrize("make,rows", [(lambda **a: cc.FusedLinear(**a), 65535 * 64),
                                       (lambda **a: cc.GroupedLinear(E=4, **a), 65535 * 64 - 4 * 63)])
def test_rows_of_a_layer_for_training(make, rows):
    """65535 blocks of 64 rows, the last of each expert with a single one; a layer that has no backward pass takes more."""
    def refused(**change):
        try:
            make(**(dict(M=rows, N=8, K=8, device=0, stream=0) | change))
        except RuntimeError as e:
            return "more blocks than a launch" in str(e)
        return False
    assert not refused() and not refused(M=rows + 1, training=False)
    assert refused(M=rows + 64)
