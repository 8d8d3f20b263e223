"""Two layers on two streams at the same time, with parts of K joined and ends of rows copied in scratch memory of their own: every pass has outputs
of its own, NaN before it, and gives the bits of that pass alone."""
import pytest
import torch

import ccglib_amd as cc
from linear_util import ACT, HALF, VT

pytestmark = pytest.mark.gpu

PASSES = 40


@pytest.mark.parametrize("shape,parts", [(3, 4), (2, 6), (4, 2)])
def test_every_pass_of_two_layers_at_once(shape, parts):
    M, N, K, t = 70, 129, 4099, VT.bfloat16
    gen = torch.Generator().manual_seed(8)
    layers = []
    for _ in range(2):
        side = torch.cuda.Stream()
        with cc.option(cc.Option.real_block, shape + 256 * parts):
            layer = cc.FusedLinear(M, N, K, 0, side.cuda_stream, t, ACT.gelu)
        layers.append((layer, [torch.randn(s, generator=gen).to(HALF[t]).cuda() for s in ((M, K), (N, K), (M, N))]))

    def outputs():
        shapes = (((M, N), HALF[t]), ((M, N), HALF[t]), ((M, K), HALF[t]), ((N, K), torch.float32), ((N,), torch.float32))
        return [torch.full(s, float("nan"), dtype=d, device="cuda") for s, d in shapes]

    def run(layer, ins, outs):
        (x, w, dy), (y, z, dx, dw, db) = ins, outs
        layer.Forward(x.data_ptr(), w.data_ptr(), 0, 0, y.data_ptr(), z.data_ptr())
        layer.Backward(dy.data_ptr(), z.data_ptr(), x.data_ptr(), w.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr())

    alone = [outputs() for _ in layers]
    at_once = [[outputs() for _ in range(PASSES)] for _ in layers]
    torch.cuda.synchronize()
    for (layer, ins), outs in zip(layers, alone):
        run(layer, ins, outs)
        torch.cuda.synchronize()
    for i in range(PASSES):
        for (layer, ins), outs in zip(layers, at_once):
            run(layer, ins, outs[i])
    torch.cuda.synchronize()
    for want, passes in zip(alone, at_once):
        assert not any(bool(v.isnan().any()) for v in want)
        for i, got in enumerate(passes):
            assert all(torch.equal(a, b) for a, b in zip(want, got)), "pass %d" % i
