"""Outputs of the 16-bit linear layers that are stored past the caches: y and z, dx, and dW of 16 and 32 bits, from 256 MiB on (y and z with
what the product reads counted in, where there is a z or a residual). Sums are short, so that a pass is all stores. Values are checked
against 64 bits on the device (bounds: linear_util.py), among NaN, at distances and addresses that are multiples of 16 bytes and at odd ones,
for the shapes whose waves write whole lines and for what the sizes choose."""
import pytest
import torch

import ccglib_amd as cc
from linear_util import ACT, HALF, TORCH, VT, backward, forward, half_step, stream

pytestmark = pytest.mark.gpu

PAST = 256 << 20
SHAPES = [0, 1, 6, 7]      # (chosen; 256 x 256, 256 x 128, 256 x 256 with the last ones cut)


def among_nan(shape, t, pitch, shift, fill=None, gen=None, scale=1.0):
    """Rows of normal values (of `fill` where that is given) `pitch` apart in a buffer of NaN."""
    rows, columns = shape
    held = torch.full((64 + shift + (rows - 1) * pitch + columns + 64,), float("nan"), dtype=t, device="cuda")
    view = held[64 + shift:].as_strided((rows, columns), (pitch, 1))
    if fill is not None:
        view.fill_(fill)
    else:
        view.copy_(torch.randn(shape, generator=gen, device="cuda") * scale)
    return view


def untouched_around(out, pitch):
    """What lies in front of, behind and between the rows of an output is NaN still."""
    rows, columns = out.shape
    at, end = out.storage_offset(), out.storage_offset() + (rows - 1) * pitch + columns
    whole = torch.empty(0, dtype=out.dtype, device="cuda").set_(out.untyped_storage())
    assert bool(whole[:at].isnan().all()) and bool(whole[end:].isnan().all())
    if pitch > columns:
        assert bool(out.as_strided((rows - 1, pitch - columns), (pitch, 1), at + columns).isnan().all())


def check(got, want, error, what):
    rel, least = half_step(got.dtype)
    worst = 0.0
    for i in range(0, got.shape[0], 1024):
        w, e = want[i:i + 1024], error[i:i + 1024]
        off = (got[i:i + 1024].double() - w).abs() - (e + rel * (w.abs() + e) + least)
        worst = max(worst, float(torch.nan_to_num(off, nan=float("inf")).max()))
    assert worst <= 0, "%s: %g more than allowed" % (what, worst)


def run(M, N, K, t, activation, odd, offsets=None, gradient_type=VT.float32, more=True, accumulate=False):
    """One forward and one backward pass. more: with z and a residual. offsets: a GroupedLinear."""
    gen = torch.Generator(device="cuda").manual_seed(M + N + K)
    E = len(offsets) - 1 if offsets else 1
    shift = 3 if odd else 0
    xp, wp, yp = ((-(-n // 8) * 8 + (5 if odd else 0)) for n in (K, K, N))
    h = HALF[t]
    x, w = among_nan((M, K), h, xp, shift, gen=gen), among_nan((E * N, K), h, wp, shift, gen=gen, scale=K ** -0.5)
    b, r = among_nan((E, N), h, N, shift, gen=gen), among_nan((M, N), h, yp, shift, gen=gen)
    dy = among_nan((M, N), h, yp, shift, gen=gen, scale=0.1)
    y, z, dx = (among_nan(s, h, p, shift, fill=77.0) for s, p in (((M, N), yp), ((M, N), yp), ((M, K), xp)))
    dw = among_nan((E * N, K), TORCH[gradient_type], wp, shift, fill=0.5)
    db = among_nan((E, N), TORCH[gradient_type], N, shift, fill=0.5)
    arguments = (N, K, 0, stream(), t, activation, gradient_type, True, xp, wp, yp)
    if offsets:
        layer = cc.GroupedLinear(E, M, *arguments)
        held = torch.tensor(offsets, dtype=torch.int32, device="cuda")
        o = (held.data_ptr(),)
    else:
        layer, o = cc.FusedLinear(M, *arguments), ()
    layer.Forward(x.data_ptr(), *o, w.data_ptr(), b.data_ptr(), r.data_ptr() if more else 0, y.data_ptr(), z.data_ptr() if more else 0)
    if not more:      # (without an activation: none is wanted)
        assert activation == ACT.none
    layer.Backward(dy.data_ptr(), z.data_ptr() if more else 0, x.data_ptr(), *o, w.data_ptr(), dx.data_ptr(), dw.data_ptr(),
                   db.data_ptr(), accumulate=accumulate)
    torch.cuda.synchronize()
    for e in range(E):
        rows, ws = slice(*offsets[e:e + 2]) if offsets else slice(0, M), slice(e * N, (e + 1) * N)
        if rows.start == rows.stop:
            assert bool((dw[ws] == (0.5 if accumulate else 0.0)).all())
            continue
        x64, w64, b64, r64, dy64 = (v.double() for v in (x[rows], w[ws], b[e], r[rows], dy[rows]))
        zw, yw, ez, ey = forward(x64, w64, b64, r64 if more else None, activation)
        check(y[rows], yw, ey, "y")
        if more:
            check(z[rows], zw, ez, "z")
        del zw, yw, ez, ey
        (dxw, dww, dbw), (edx, edw, edb) = backward(dy64, z[rows].double() if more else dy64, x64, w64, activation, h)
        check(dx[rows], dxw, edx, "dx")
        if accumulate:
            dww, dbw = dww + 0.5, dbw + 0.5
            edw, edb = edw + 2.0 ** -23 * dww.abs(), edb + 2.0 ** -23 * dbw.abs()
        check(dw[ws], dww, edw, "dw")
        check(db[e:e + 1], dbw[None], edb[None], "db")
        del dxw, dww, edx, edw
    if offsets:
        for out in (y, dx) + ((z,) if more else ()):
            assert bool((out[:offsets[0]] == 77.0).all()) and bool((out[offsets[E]:] == 77.0).all()), "rows of no expert"
    for out, pitch in ((y, yp), (dx, xp), (dw, wp), (z, yp)):
        untouched_around(out, pitch)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("t", list(HALF))
def test_y_and_z_with_a_residual(t, odd, shape):
    M, N, K = 4100, 16400, 72
    assert 2 * 3 * M * N >= PAST > 2 * 2 * M * K
    with cc.option(cc.Option.real_block, shape):
        run(M, N, K, t, ACT.silu, odd)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("odd", [False, True])
def test_y_alone(odd, shape):
    M, N, K = 8200, 16400, 40
    assert 2 * M * N >= PAST
    with cc.option(cc.Option.real_block, shape):
        run(M, N, K, VT.bfloat16, ACT.none, odd, more=False)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("odd", [False, True])
def test_dx(odd, shape):
    M, N, K = 8200, 40, 16400
    assert 2 * M * K >= PAST
    with cc.option(cc.Option.real_block, shape):
        run(M, N, K, VT.float16, ACT.gelu, odd)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("N,K,gradient_type,accumulate", [(8200, 16400, VT.bfloat16, False), (8200, 8200, VT.float32, False),
                                                          (8200, 8200, VT.float32, True)])
def test_dw(N, K, gradient_type, accumulate, odd, shape):
    assert (4 if gradient_type == VT.float32 else 2) * N * K >= PAST
    with cc.option(cc.Option.real_block, shape):
        run(40, N, K, VT.bfloat16, ACT.none, odd, gradient_type=gradient_type, accumulate=accumulate)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("odd", [False, True])
def test_experts(odd, shape):
    """y, z and dx of rows in front of, of and behind three experts, one of which has none; then dW of four."""
    with cc.option(cc.Option.real_block, shape):
        run(4200, 16400, 72, VT.bfloat16, ACT.silu, odd, offsets=[5, 1900, 1900, 4195])
        run(8300, 40, 16400, VT.bfloat16, ACT.relu, odd, offsets=[5, 3900, 3900, 8295])
        assert 4 * 4 * 4100 * 4100 >= PAST
        run(200, 4100, 4100, VT.float16, ACT.none, odd, offsets=[3, 20, 20, 120, 199], accumulate=odd)
