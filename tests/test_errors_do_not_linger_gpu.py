"""An object that cannot be created, for want of memory, says so; the calls behind it, of other objects, do not."""
import pytest
import torch

import ccglib_amd as cc
from scaled_util import stream

pytestmark = pytest.mark.gpu
VT = cc.ValueType


def fails():
    with pytest.raises(RuntimeError, match="out of memory"):
        cc.Orthogonalize(60, 100000, 100000, 0, stream(), VT.float32)     # (terabytes)


def test_runs_behind_a_failed_creation():
    x = torch.randn((40, 64), device="cuda")
    q, s = torch.zeros((40, 64), dtype=torch.uint8, device="cuda"), torch.zeros((1, 48), device="cuda")
    c, out = torch.zeros((40, 40), device="cuda"), torch.zeros_like(x)
    p = [t.data_ptr() for t in (x, q, s, c, out)]
    quantize = cc.Quantize(1, 40, 64, 0, stream(), VT.float32)
    product = cc.ScaledGEMM(1, 40, 40, 64, 0, stream(), c_type=VT.float32, b_group=cc.ScaleGroup.rows)
    layer = cc.ScaledLinear(40, 64, 64, 0, stream(), VT.float32)
    update = cc.Orthogonalize(1, 40, 64, 0, stream(), VT.float32)
    w = torch.randn((64, 64), device="cuda")
    packing = cc.Packing(4096, cc.Direction.forward, 0, stream())
    bits, packed = torch.ones(4096, dtype=torch.uint8, device="cuda"), torch.zeros(512, dtype=torch.uint8, device="cuda")
    for run in (lambda: quantize.Run(p[0], p[1], p[2]), lambda: product.Run(p[1], p[2], p[1], p[2], p[3]),
                lambda: layer.SetWeights(w.data_ptr()), lambda: layer.Forward(p[0], p[4]), lambda: update.Run(p[0], p[4]),
                lambda: packing.Run(bits.data_ptr(), packed.data_ptr())):
        fails()
        run()
        torch.cuda.synchronize()
    assert bool(c.ne(0).any()) and bool(out.ne(0).any()) and bool((packed == 255).all())


def test_a_creation_behind_a_failed_one():
    fails()
    layer = cc.ScaledLinear(40, 64, 64, 0, stream(), VT.float32)
    w = torch.randn((64, 64), device="cuda")
    layer.SetWeights(w.data_ptr())
    torch.cuda.synchronize()
