"""The names of a layer's kernels: where dx and dW are small enough to be one launch, the names say so."""
import pytest

import ccglib_amd as cc
from linear_util import stream

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("make", [lambda *s: cc.FusedLinear(*s, 0, stream()), lambda *s: cc.GroupedLinear(2, *s, 0, stream())])
def test_gradients_in_one_launch(make):
    small, large = make(100, 100, 100), make(5000, 4000, 4000)
    for product in (1, 2):
        assert small.KernelName(product).startswith("gemm_linear_backward<bfloat16, ")
        assert small.KernelName(product).endswith("in one launch")
        assert large.KernelName(product).startswith("gemm_linear<bfloat16, ") and "one launch" not in large.KernelName(product)
    assert "one launch" not in small.KernelName() + large.KernelName()


def test_forward_only():
    layer = cc.FusedLinear(100, 100, 100, 0, stream(), training=False)
    assert "one launch" not in layer.KernelName()
    with pytest.raises(RuntimeError, match="no such product"):
        layer.KernelName(1)
