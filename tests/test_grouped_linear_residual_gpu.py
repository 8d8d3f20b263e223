"""GroupedLinear with a residual: y and z of every expert against 64 bits (bounds: linear_util.py), for every block shape and the kernel for a few
rows; residuals of rows of no expert are not read; y may be the residual."""
import math

import pytest
import torch

import ccglib_amd as cc
from linear_util import ACT, HALF, VT, among_nan, check, forward, stream

pytestmark = pytest.mark.gpu


def run(E, M, N, K, t, activation, offsets, pitches=(0, 0, 0), shift=0, bias=True):
    gen = torch.Generator().manual_seed(E + M + 7 * N + 11 * K)
    xp, wp, yp = pitches

    def normal(rows, columns, scale=1.0):
        return (torch.randn((rows, columns), generator=gen, dtype=torch.float64) * scale).to(HALF[t])
    x, w, b, r = normal(M, K), normal(E * N, K, max(1, K) ** -0.5), normal(E, N), normal(M, N)
    mine = torch.zeros(M, dtype=torch.bool)
    mine[offsets[0]:offsets[E]] = True
    x[~mine], r[~mine] = math.nan, math.nan             # (rows of no expert: not read)
    xd, wd, bd, rd = among_nan(x, xp, shift), among_nan(w, wp, shift), among_nan(b), among_nan(r, yp, shift)
    y, z = (among_nan(torch.full((M, N), 77.0, dtype=HALF[t]), yp, shift) for _ in range(2))
    o = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    layer = cc.GroupedLinear(E, M, N, K, 0, stream(), t, activation, training=False, x_pitch=xp, w_pitch=wp, y_pitch=yp)
    arguments = (xd.data_ptr(), o.data_ptr(), wd.data_ptr(), bd.data_ptr() if bias else 0, rd.data_ptr())
    layer.Forward(*arguments, y.data_ptr(), z.data_ptr())
    torch.cuda.synchronize()
    for e in range(E):
        rows = slice(offsets[e], offsets[e + 1])
        x64, w64, b64, r64 = (v.double().cuda() for v in (x[rows], w[e * N:(e + 1) * N], b[e], r[rows]))
        zw, yw, ez, ey = forward(x64, w64, b64 if bias else None, r64, activation)
        check(z[rows], zw, ez, "z of %d" % e)
        check(y[rows], yw, ey, "y of %d" % e)
    for out in (y, z):
        assert bool((out[~mine.cuda()] == 77.0).all()), "rows of no expert"
    # in place: the same bits, and NaN stays where it was
    layer.Forward(*arguments, rd.data_ptr(), z.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(rd[mine.cuda()], y[mine.cuda()]) and bool(rd[~mine.cuda()].isnan().all())
    return layer


@pytest.mark.parametrize("shape", range(0, 8))
@pytest.mark.parametrize("pitches,shift", [((584, 584, 264), 0), ((579, 581, 257), 1)])
def test_every_shape(shape, pitches, shift):
    with cc.option(cc.Option.real_block, shape):
        run(3, 700, 255, 577, VT.bfloat16, ACT.gelu, [4, 290, 290, 690], pitches=pitches, shift=shift)
        run(9, 100, 24, 136, VT.float16, ACT.none, [0, 1, 3, 3, 40, 41, 70, 90, 98, 100], bias=False)


@pytest.mark.parametrize("offsets", [[0, 2, 2, 30], [3, 3, 3, 29], [0, 30, 30, 30]])
@pytest.mark.parametrize("K", [40, 1031])
def test_few_rows(offsets, K):
    layer = run(3, 30, 33, K, VT.bfloat16, ACT.silu, offsets, pitches=(K + 1, K, 35), shift=1)
    assert "linear_rows" in layer.KernelName()
