"""ScaledLinear: dx is that of the W of the last Forward, or refused."""
import pytest
import torch

import ccglib_amd as cc
from scaled_util import stream

pytestmark = pytest.mark.gpu
VT = cc.ValueType


def test_weights_set_between_forward_and_backward():
    M, N, K = 5, 40, 70
    gen = torch.Generator().manual_seed(1)
    x, w, dy = (torch.randn(s, generator=gen).cuda() for s in ((M, K), (N, K), (M, N)))
    twice = 2 * w
    y, dx, dw = torch.empty((M, N), device="cuda"), torch.empty((M, K), device="cuda"), torch.empty((N, K), device="cuda")
    layer = cc.ScaledLinear(M, N, K, 0, stream(), VT.float32)
    layer.SetWeights(w.data_ptr())
    layer.Forward(x.data_ptr(), y.data_ptr())
    layer.Backward(dy.data_ptr(), dx.data_ptr(), dw.data_ptr())
    torch.cuda.synchronize()
    want_dx, want_dw = dx.clone(), dw.clone()
    layer.SetWeights(twice.data_ptr())
    dx.fill_(7.0)
    for d_dw in (0, dw.data_ptr()):
        with pytest.raises(RuntimeError, match="weights were set since"):
            layer.Backward(dy.data_ptr(), dx.data_ptr(), d_dw)
    dw.fill_(7.0)
    layer.Backward(dy.data_ptr(), 0, dw.data_ptr())          # (x is still that of the forward)
    torch.cuda.synchronize()
    assert bool((dx == 7).all()) and torch.equal(dw, want_dw)
    layer.Forward(x.data_ptr(), y.data_ptr())
    layer.Backward(dy.data_ptr(), dx.data_ptr(), dw.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(dx, 2 * want_dx) and torch.equal(dw, want_dw)
