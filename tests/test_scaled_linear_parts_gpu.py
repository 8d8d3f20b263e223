"""ScaledLinear where its products cut K into parts and have unlike numbers of blocks: every step of one object writes all of y,
dx and dW, and the same bits each time. Against products in 64 bits, within the bounds of test_scaled_gemm_gpu.py."""
import pytest
import torch

import ccglib_amd as cc
from scaled_util import WIDE, stream
from test_scaled_linear_gpu import near, through

pytestmark = pytest.mark.gpu
VT, SG, ST = cc.ValueType, cc.ScaleGroup, cc.ScaleType


def steps(M, N, K, t, st, tg=VT.float8e5m2, count=2):
    gen = torch.Generator().manual_seed(M + N)
    x = torch.randn((M, K), generator=gen).to(WIDE[t]).cuda()
    w = (torch.randn((N, K), generator=gen) / K ** 0.5).to(WIDE[t]).cuda()
    dy = (torch.randn((M, N), generator=gen) * 0.01).to(WIDE[t]).cuda()
    y, dx = torch.empty((M, N), dtype=WIDE[t], device="cuda"), torch.empty((M, K), dtype=WIDE[t], device="cuda")
    dw = torch.empty((N, K), device="cuda")
    layer = cc.ScaledLinear(M, N, K, 0, stream(), t, tg, st)
    kept = []
    for _ in range(count):
        for out in (y, dx, dw):
            out.fill_(float("nan"))
        layer.SetWeights(w.data_ptr())
        layer.Forward(x.data_ptr(), y.data_ptr())
        layer.Backward(dy.data_ptr(), dx.data_ptr(), dw.data_ptr())
        torch.cuda.synchronize()
        kept.append((y.clone(), dx.clone(), dw.clone()))
    e4 = VT.float8e4m3
    assert near(y, through(x, e4, SG.rows, st), through(w, e4, SG.blocks, st), t)
    assert near(dx, through(dy, tg, SG.rows, st), through(w.t(), e4, SG.blocks, st), t)
    assert near(dw, through(dy.t(), tg, SG.rows, st), through(x.t(), e4, SG.rows, st), VT.float32)
    for later in kept[1:]:
        assert all(torch.equal(a, b) for a, b in zip(kept[0], later))
    # dW added to, the next step's forward behind it
    total = torch.ones_like(dw)
    layer.Backward(dy.data_ptr(), 0, total.data_ptr(), accumulate_dw=True)
    y.fill_(float("nan"))
    layer.Forward(x.data_ptr(), y.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(total, dw + 1.0) and torch.equal(y, kept[0][0])


@pytest.mark.parametrize("M,N,K,t,st", [
    (32, 2560, 5120, VT.float32, ST.float32), (32, 5120, 2560, VT.float32, ST.float32), (16, 4096, 8192, VT.float32, ST.float32),
    (2649, 127, 5376, VT.bfloat16, ST.float32), (180, 4441, 6379, VT.float32, ST.e8m0)])
def test_layers_that_split_by_default(M, N, K, t, st):
    steps(M, N, K, t, st)


@pytest.mark.parametrize("t", list(WIDE))
@pytest.mark.parametrize("st", list(ST))
@pytest.mark.parametrize("shape,parts", [(2, 3), (3, 2), (4, 5), (5, 3)])
def test_every_block_shape_in_parts(t, st, shape, parts):
    with cc.option(cc.Option.real_block, shape + 256 * parts):
        steps(140, 1100, 2300, t, st)
        steps(900, 70, 1300, t, st)
