"""ScaledLinear: y, dx and dW against products in 64 bits of the 8-bit copies that Quantize's formula gives, within the
bounds of the products (test_scaled_gemm_gpu.py); dx and dW against differences of the loss where every value is one that
8 bits hold, so that the layer is the linear function itself."""
import itertools

import pytest
import torch

import ccglib_amd as cc
from scaled_util import F8, WIDE, quantized, stream, values_of
from test_scaled_gemm_gpu import bound

pytestmark = pytest.mark.gpu
VT, SG, ST = cc.ValueType, cc.ScaleGroup, cc.ScaleType


def through(x, vtype, group, st):
    return values_of(*quantized(x[None], vtype, group, st), group)[0].cuda()


def near(got, a, b, ctype, extra=None):
    """got against a b^T"""
    want, S = a @ b.t().contiguous(), a.abs() @ b.abs().t().contiguous()
    if extra is not None:
        want, S = want + extra.double(), S + extra.double().abs()
    return bool(((got.double() - want).abs() <= bound(want, S, a.shape[1], ctype)).all())


@pytest.mark.parametrize("t,tg", list(itertools.product(WIDE, F8)))
@pytest.mark.parametrize("st", list(ST))
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (5, 130, 257), (300, 255, 576), (129, 64, 40)])
def test_forward_and_backward(t, tg, st, M, N, K):
    gen = torch.Generator().manual_seed(M + N)
    x = torch.randn((M, K), generator=gen).to(WIDE[t]).cuda()
    w = (torch.randn((N, K), generator=gen) / K ** 0.5).to(WIDE[t]).cuda()
    dy = (torch.randn((M, N), generator=gen) * 0.01).to(WIDE[t]).cuda()
    y, dx = torch.empty((M, N), dtype=WIDE[t], device="cuda"), torch.empty((M, K), dtype=WIDE[t], device="cuda")
    dw = torch.empty((N, K), device="cuda")
    layer = cc.ScaledLinear(M, N, K, 0, stream(), t, tg, st)
    layer.SetWeights(w.data_ptr())
    layer.Forward(x.data_ptr(), y.data_ptr())
    layer.Backward(dy.data_ptr(), dx.data_ptr(), dw.data_ptr())
    torch.cuda.synchronize()
    e4 = VT.float8e4m3
    assert near(y, through(x, e4, SG.rows, st), through(w, e4, SG.blocks, st), t)
    assert near(dx, through(dy, tg, SG.rows, st), through(w.t(), e4, SG.blocks, st), t)
    gy, gx = through(dy.t(), tg, SG.rows, st), through(x.t(), e4, SG.rows, st)
    assert near(dw, gy, gx, VT.float32)
    # either gradient alone, and dW added to
    again = torch.empty_like(dx)
    layer.Backward(dy.data_ptr(), again.data_ptr(), 0)
    old = torch.randn((N, K), generator=gen).cuda()
    total = old.clone()
    layer.Backward(dy.data_ptr(), 0, total.data_ptr(), accumulate_dw=True)
    torch.cuda.synchronize()
    assert torch.equal(again, dx)
    assert near(total, gy, gx, VT.float32, extra=old)
    # forward only
    serving = cc.ScaledLinear(M, N, K, 0, stream(), t, tg, st, training=False)
    serving.SetWeights(w.data_ptr())
    other = torch.empty_like(y)
    serving.Forward(x.data_ptr(), other.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(other, y)
    with pytest.raises(RuntimeError, match="without training"):
        serving.Backward(dy.data_ptr(), dx.data_ptr(), dw.data_ptr())


@pytest.mark.parametrize("tg", list(F8))
@pytest.mark.parametrize("st", list(ST))
def test_gradients_are_the_differences_of_the_loss(tg, st):
    """Every group's largest value is 7 (448 is 7 * 2^6, 57344 is 7 * 2^13), so scales are powers of two and small integers
    pass as they are: the loss sum(dy * y) is exactly linear in x and in W, and its differences over a step of 1 are the
    gradients, exactly (sums of integers below 2^24)."""
    M, N, K = 6, 130, 140
    gen = torch.Generator().manual_seed(9)

    def whole(rows, cols):
        v = torch.randint(-3, 4, (rows, cols), generator=gen).float()
        v[:, ::128] = 7.0          # in every group of a row, and of a column
        v[::128, :] = 7.0
        return v.cuda()
    x, w, dy = whole(M, K), whole(N, K), whole(M, N)
    layer = cc.ScaledLinear(M, N, K, 0, stream(), VT.float32, tg, st)
    y, dx, dw = torch.empty((M, N), device="cuda"), torch.empty((M, K), device="cuda"), torch.empty((N, K), device="cuda")

    def loss(x, w):
        layer.SetWeights(w.data_ptr())
        layer.Forward(x.data_ptr(), y.data_ptr())
        torch.cuda.synchronize()
        return float((y.double() * dy.double()).sum())
    base = loss(x, w)
    layer.Backward(dy.data_ptr(), dx.data_ptr(), dw.data_ptr())
    torch.cuda.synchronize()
    want_dx, want_dw = dy.double() @ w.double(), dy.double().t().contiguous() @ x.double()
    assert torch.equal(dx.double(), want_dx) and torch.equal(dw.double(), want_dw)
    for m, k in [(1, 1), (5, 139), (3, 70)]:
        moved = x.clone()
        moved[m, k] += 1.0
        assert loss(moved, w) - base == float(dx[m, k])
    for n, k in [(1, 1), (129, 139), (64, 127)]:
        moved = w.clone()
        moved[n, k] += 1.0
        assert loss(x, moved) - base == float(dw[n, k])


def test_order_of_calls():
    t = torch.zeros(4096, device="cuda")
    layer = cc.ScaledLinear(4, 4, 4, 0, stream(), VT.float32)
    with pytest.raises(RuntimeError, match="before the weights were set"):
        layer.Forward(t.data_ptr(), t.data_ptr())
    layer.SetWeights(t.data_ptr())
    with pytest.raises(RuntimeError, match="backward before forward"):
        layer.Backward(t.data_ptr(), t.data_ptr(), t.data_ptr())
    with pytest.raises(RuntimeError, match="null pointer"):
        layer.Forward(0, t.data_ptr())
    with pytest.raises(RuntimeError, match="misaligned"):
        layer.SetWeights(t.data_ptr() + 2)
    with pytest.raises(RuntimeError, match="null pointer"):
        layer.SetWeights(0)
