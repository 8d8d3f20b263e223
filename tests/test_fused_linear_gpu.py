"""FusedLinear: y, z, dx, dW and dbias against 64 bits, within the bounds that linear_util.py derives: types, activations, every
block shape and parts of K, sizes that fit no tile, rows at odd distances and addresses among NaN, empty extents, values that are
not finite, and gradients against differences."""
import itertools
import math

import pytest
import torch

import ccglib_amd as cc
from linear_util import ACT, HALF, TORCH, VT, among_nan, act, act_gradient, backward, check, forward, stream

pytestmark = pytest.mark.gpu


def made(gen, rows, columns, t, scale=1.0):
    return (torch.randn((rows, columns), generator=gen, dtype=torch.float64) * scale).to(HALF[t])


def run_layer(M, N, K, t, activation, gradient_type=VT.float32, pitches=(0, 0, 0), shift=0, bias=True, residual=True, seed=0,
              accumulate=False):
    """One forward and one backward pass, both checked."""
    gen = torch.Generator().manual_seed(seed + M + 7 * N + 11 * K)
    x, w = made(gen, M, K, t), made(gen, N, K, t, max(1, K) ** -0.5)
    b, r, dy = made(gen, 1, N, t), made(gen, M, N, t), made(gen, M, N, t, 0.1)
    xp, wp, yp = pitches

    def there(v, pitch):
        return among_nan(v, pitch or None, shift)

    def room(rows, columns, dtype, pitch):
        return among_nan(torch.full((rows, columns), math.nan, dtype=dtype), pitch or None, shift)
    dev = {"x": there(x, xp), "w": there(w, wp), "b": there(b, 0), "r": there(r, yp), "dy": there(dy, yp)}
    y, z, dx = room(M, N, HALF[t], yp), room(M, N, HALF[t], yp), room(M, K, HALF[t], xp)
    layer = cc.FusedLinear(M, N, K, 0, stream(), t, activation, gradient_type, True, xp, wp, yp)
    layer.Forward(dev["x"].data_ptr(), dev["w"].data_ptr(), dev["b"].data_ptr() if bias else 0,
                  dev["r"].data_ptr() if residual else 0, y.data_ptr(), z.data_ptr())
    torch.cuda.synchronize()
    x64, w64, b64, r64, dy64 = (v.double().cuda() for v in (x, w, b[0], r, dy))
    zw, yw, ez, ey = forward(x64, w64, b64 if bias else None, r64 if residual else None, activation)
    check(z, zw, ez, "z")
    check(y, yw, ey, "y")
    old_w, old_b = made(gen, N, K, t), made(gen, 1, N, t)
    dw = among_nan(old_w.to(TORCH[gradient_type]), wp or None, shift)
    db = among_nan(old_b.to(TORCH[gradient_type]), None, shift)
    layer.Backward(dev["dy"].data_ptr(), z.data_ptr() if activation != ACT.none else 0, dev["x"].data_ptr(), dev["w"].data_ptr(),
                   dx.data_ptr(), dw.data_ptr(), db.data_ptr(), accumulate=accumulate)
    torch.cuda.synchronize()
    (dxw, dww, dbw), (edx, edw, edb) = backward(dy64, z.double(), x64, w64, activation, HALF[t])
    if accumulate:
        dww, dbw = dww + old_w.cuda().double(), dbw + old_b.cuda().double()[0]
        edw, edb = edw + 2.0 ** -23 * dww.abs(), edb + 2.0 ** -23 * dbw.abs()
    check(dx, dxw, edx, "dx")
    check(dw, dww, edw, "dw")
    check(db[0], dbw, edb, "db")
    # what lies between the rows of an output is left alone
    for out, pitch in ((y, yp), (z, yp), (dx, xp), (dw, wp)):
        if pitch and out.shape[0] > 1 and pitch > out.shape[1]:
            between = out.as_strided((out.shape[0] - 1, pitch - out.shape[1]), (pitch, 1), out.storage_offset() + out.shape[1])
            assert bool(between.isnan().all())
    return layer


SIZES = [(1, 1, 1), (3, 2, 5), (64, 64, 64), (5, 130, 257), (129, 64, 40), (17, 8, 7), (40, 3, 200), (300, 255, 577), (257, 520, 136)]


@pytest.mark.parametrize("t,activation", list(itertools.product(HALF, ACT)))
@pytest.mark.parametrize("M,N,K", SIZES)
def test_forward_and_backward(t, activation, M, N, K):
    run_layer(M, N, K, t, activation)


@pytest.mark.parametrize("t", list(HALF))
@pytest.mark.parametrize("shape,parts", [(s, p) for s in range(1, 7) for p in (1, 3)])
@pytest.mark.parametrize("M,N,K", [(300, 261, 713), (33, 600, 64), (512, 256, 1000)])
def test_every_shape(t, shape, parts, M, N, K):
    with cc.option(cc.Option.real_block, shape + 256 * parts):
        layer = run_layer(M, N, K, t, ACT.silu)
    assert "K in" in layer.KernelName(2)


@pytest.mark.parametrize("shape", range(1, 7))
@pytest.mark.parametrize("K", [1, 2, 7, 8, 9, 15, 63, 64, 65, 71, 72, 120, 127, 128, 129, 191, 193, 256, 449])
def test_every_length_of_the_sum(shape, K):
    """K is the sum's length of y, N of dx, M of dW."""
    with cc.option(cc.Option.real_block, shape):
        run_layer(40, 24, K, VT.bfloat16, ACT.none)
        run_layer(40, K, 24, VT.float16, ACT.none)
        run_layer(K, 40, 24, VT.bfloat16, ACT.none)


@pytest.mark.parametrize("shape", range(0, 7))
@pytest.mark.parametrize("pitches,shift", [((584, 584, 264), 0), ((584, 584, 264), 1), ((577, 577, 255), 3), ((579, 581, 257), 0),
                                           ((1000, 600, 400), 5)])
def test_distances_and_addresses(shape, pitches, shift):
    with cc.option(cc.Option.real_block, shape):
        run_layer(70, 255, 577, VT.bfloat16, ACT.gelu, pitches=pitches, shift=shift)
        run_layer(9, 3, 5, VT.float16, ACT.none, pitches=(8, 8, 8), shift=shift)
        run_layer(9, 3, 5, VT.float16, ACT.relu, pitches=(5, 6, 7), shift=shift)


@pytest.mark.parametrize("t", list(HALF))
@pytest.mark.parametrize("gradient_type,accumulate", [(VT.float32, False), (VT.float32, True), (None, False)])
def test_gradients_of_weights_in_either_type(t, gradient_type, accumulate):
    run_layer(130, 70, 90, t, ACT.none, gradient_type or t, accumulate=accumulate)
    run_layer(130, 70, 90, t, ACT.silu, gradient_type or t, accumulate=accumulate, bias=False, residual=False)


def test_long_sums_and_many_rows():
    run_layer(16, 48, 9000, VT.bfloat16, ACT.none)
    run_layer(5000, 33, 48, VT.float16, ACT.relu)


@pytest.mark.parametrize("M,N,K", [(0, 5, 6), (5, 0, 6), (5, 6, 0), (0, 0, 0), (0, 40, 0)])
def test_empty_extents(M, N, K):
    run_layer(M, N, K, VT.bfloat16, ACT.gelu)


def test_the_same_bits_every_time_and_single_outputs():
    M, N, K, t = 200, 300, 500, VT.bfloat16
    gen = torch.Generator().manual_seed(3)
    x, w, dy, z = (made(gen, *s, t).cuda() for s in ((M, K), (N, K), (M, N), (M, N)))
    layer = cc.FusedLinear(M, N, K, 0, stream(), t, ACT.gelu)

    def outputs(dx_wanted=True, dw_wanted=True, db_wanted=True):
        y, dx = torch.zeros_like(dy), torch.zeros_like(x)
        dw, db = torch.zeros((N, K), device="cuda"), torch.zeros(N, device="cuda")
        layer.Forward(x.data_ptr(), w.data_ptr(), 0, 0, y.data_ptr())
        layer.Backward(dy.data_ptr(), z.data_ptr(), x.data_ptr(), w.data_ptr(), dx.data_ptr() if dx_wanted else 0,
                       dw.data_ptr() if dw_wanted else 0, db.data_ptr() if db_wanted else 0)
        torch.cuda.synchronize()
        return y, dx, dw, db
    all_of_them = outputs()
    for wanted in itertools.product((True, False), repeat=3):
        for i, (got, want) in enumerate(zip(outputs(*wanted), all_of_them)):
            assert torch.equal(got, want if i == 0 or wanted[i - 1] else torch.zeros_like(want))


def test_y_may_be_the_residual():
    M, N, K = 70, 90, 300
    gen = torch.Generator().manual_seed(4)
    x, w, r = (made(gen, *s, VT.float16).cuda() for s in ((M, K), (N, K), (M, N)))
    layer = cc.FusedLinear(M, N, K, 0, stream(), VT.float16, ACT.silu, training=False)
    y = torch.empty_like(r)
    layer.Forward(x.data_ptr(), w.data_ptr(), 0, r.data_ptr(), y.data_ptr())
    layer.Forward(x.data_ptr(), w.data_ptr(), 0, r.data_ptr(), r.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(y, r)


@pytest.mark.parametrize("activation", list(ACT))
def test_values_that_are_not_finite(activation):
    """A NaN or an infinity in a row of x or W shows in its row and column of y, and nowhere else."""
    M, N, K, t = 40, 50, 73, VT.bfloat16
    gen = torch.Generator().manual_seed(5)
    x, w = made(gen, M, K, t), made(gen, N, K, t, 0.1)
    x[7, 72], x[9, 0], w[11, 72], x[30, 3] = math.nan, math.inf, math.nan, -math.inf
    y = torch.zeros((M, N), dtype=HALF[t], device="cuda")
    layer = cc.FusedLinear(M, N, K, 0, stream(), t, activation, training=False)
    xd, wd = x.cuda(), w.cuda()
    layer.Forward(xd.data_ptr(), wd.data_ptr(), 0, 0, y.data_ptr())
    torch.cuda.synchronize()
    want = act(x.double() @ w.double().t(), activation)
    got = y.double().cpu()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    assert torch.equal(got[got.isinf()], want[want.isinf()])
    # gradients: far out on either side act' is 0 or 1, whatever a' is
    z = torch.tensor([[-3e38, -1e20, -300.0, -40.0, 0.0, 40.0, 300.0, 1e20, 3e38, math.nan]]).to(HALF[t]).cuda()
    dy, db = torch.ones_like(z), torch.zeros(10, device="cuda")
    cc.FusedLinear(1, 10, 8, 0, stream(), t, activation).Backward(dy.data_ptr(), z.data_ptr(), 0, 0, 0, 0, db.data_ptr())
    torch.cuda.synchronize()
    half = {ACT.none: 1.0, ACT.relu: 0.0}.get(activation, 0.5)
    low, nan = (1.0, 1.0) if activation == ACT.none else (0.0, 0.0 if activation == ACT.relu else math.nan)
    want = torch.tensor([low] * 4 + [half] + [1.0] * 4 + [nan])
    assert torch.allclose(db.cpu(), want, atol=1e-15, rtol=0.0, equal_nan=True)


@pytest.mark.parametrize("activation", [ACT.gelu, ACT.silu])
def test_the_activations_gradient_is_its_difference(activation):
    """dbias of one row of ones is act'(z): against a central difference of act over 2 h = 2^-9, which a third derivative of
    at most 3 moves by h^2 / 6 * 3 < 2e-6, next to the error that act_gradient_error derives (below 1e-5 here)."""
    z = torch.linspace(-9, 9, 500).to(torch.bfloat16)
    dy, db = torch.ones_like(z).cuda(), torch.zeros(500, device="cuda")
    zd = z.cuda()
    cc.FusedLinear(1, 500, 8, 0, stream(), VT.bfloat16, activation).Backward(dy.data_ptr(), zd.data_ptr(), 0, 0, 0, 0, db.data_ptr())
    torch.cuda.synchronize()
    h, v = 2.0 ** -10, z.double()
    difference = (act(v + h, activation) - act(v - h, activation)) / (2 * h)
    assert float((db.cpu().double() - difference).abs().max()) < 1.2e-5
    assert float((act_gradient(v, activation) - difference).abs().max()) < 2e-6


def test_gradients_are_the_differences_of_the_loss():
    """Small whole numbers: the loss sum(dy * y) is exactly linear in x, W and bias, and its differences over a step of 1 are the
    gradients (sums below 2^24; y below 2^11 is exact in float16)."""
    M, N, K, t = 6, 130, 140, VT.float16
    gen = torch.Generator().manual_seed(9)

    def whole(rows, columns):
        return torch.randint(-1, 2, (rows, columns), generator=gen).to(torch.float16).cuda()
    x, w, dy, b = whole(M, K), whole(N, K), whole(M, N), whole(1, N)
    layer = cc.FusedLinear(M, N, K, 0, stream(), t)
    y, dx = torch.empty((M, N), dtype=torch.float16, device="cuda"), torch.empty_like(x)
    dw, db = torch.empty((N, K), device="cuda"), torch.empty(N, device="cuda")

    def loss(x, w, b):
        layer.Forward(x.data_ptr(), w.data_ptr(), b.data_ptr(), 0, y.data_ptr())
        torch.cuda.synchronize()
        return float((y.double() * dy.double()).sum())
    base = loss(x, w, b)
    layer.Backward(dy.data_ptr(), 0, x.data_ptr(), w.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr())
    torch.cuda.synchronize()
    for m, k in [(1, 1), (5, 139), (3, 70)]:
        moved = x.clone()
        moved[m, k] += 1.0
        assert loss(moved, w, b) - base == float(dx[m, k])
    for n, k in [(1, 1), (129, 139), (64, 127)]:
        moved = w.clone()
        moved[n, k] += 1.0
        assert loss(x, moved, b) - base == float(dw[n, k])
    for n in (0, 77, 129):
        moved = b.clone()
        moved[0, n] += 1.0
        assert loss(x, w, moved) - base == float(db[n])


def test_refusals_of_a_run():
    t = torch.zeros(4096, dtype=torch.bfloat16, device="cuda")
    p = t.data_ptr()
    layer = cc.FusedLinear(4, 4, 4, 0, stream(), activation=ACT.gelu, gradient_type=VT.bfloat16)
    for args, message in [((0, p, 0, 0, p), "x"), ((p, 0, 0, 0, p), "weights"), ((p, p, 0, 0, 0), "y")]:
        with pytest.raises(RuntimeError, match="null pointer: FusedLinear, " + message):
            layer.Forward(*args)
    for i in range(6):
        args = [p] * 6
        args[i] = p + 1
        with pytest.raises(RuntimeError, match="misaligned"):
            layer.Forward(*args)
    for args, message in [((0, p, p, p, p, p), "dy"), ((p, 0, p, p, p, p), "z"), ((p, p, 0, p, p, p), "x"), ((p, p, p, 0, p, p), "weights")]:
        with pytest.raises(RuntimeError, match="null pointer: FusedLinear, " + message):
            layer.Backward(*args)
    with pytest.raises(RuntimeError, match="added to are float32"):
        layer.Backward(p, p, p, p, p, p, p, accumulate=True)
    with pytest.raises(RuntimeError, match="without training"):
        cc.FusedLinear(4, 4, 4, 0, stream(), training=False).Backward(p, p, p, p, p, p)
    with pytest.raises(RuntimeError, match="no such product"):
        layer.KernelName(3)


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 33])
@pytest.mark.parametrize("N,K", [(1, 1), (15, 31), (16, 32), (17, 33), (40, 255), (33, 1024), (50, 1031), (64, 1800), (100, 2048)])
def test_few_rows(M, N, K):
    """The kernel for a few rows: whole steps of K or none, and what is left of it, at even and odd distances."""
    layer = run_layer(M, N, K, VT.bfloat16, ACT.gelu, pitches=(K + M % 3, K + M % 2, N + M % 5), shift=M % 2)
    run_layer(M, N, K, VT.float16, ACT.none, bias=False, residual=False)
    assert "linear_rows" in layer.KernelName()


@pytest.mark.parametrize("M,N,K", [(600, 600, 72), (8, 600, 1030)])
def test_operands_beyond_32_bits(M, N, K):
    """Rows 8 MiB apart: 5 GB of W, and of x, y, z and their gradients where there are 600 rows."""
    run_layer(M, N, K, VT.bfloat16, ACT.gelu, pitches=(1 << 22,) * 3)


def test_weights_that_are_the_last_row_of_x():
    """The two end together and are of different lengths. Small whole numbers: sums are exact."""
    M, N, K = 3, 1, 2
    x = torch.tensor([[1, 2], [3, 4], [5, 6]], dtype=torch.bfloat16, device="cuda")
    dy = torch.tensor([[1], [10], [100]], dtype=torch.bfloat16, device="cuda")
    y, dx, dw = torch.empty_like(dy), torch.empty_like(x), torch.empty((N, K), device="cuda")
    layer = cc.FusedLinear(M, N, K, 0, stream())
    w = x.data_ptr() + 2 * (M - 1) * K
    layer.Forward(x.data_ptr(), w, 0, 0, y.data_ptr())
    layer.Backward(dy.data_ptr(), 0, x.data_ptr(), w, dx.data_ptr(), dw.data_ptr())
    torch.cuda.synchronize()
    assert y.flatten().tolist() == [17, 39, 61]
    assert dx.tolist() == [[5, 6], [50, 60], [500, 600]] and dw.tolist() == [[531, 642]]


@pytest.mark.parametrize("t", list(HALF))
@pytest.mark.parametrize("rows,columns,rest", [(4000, 5100, 64), (3900, 6100, 128), (5000, 6100, 224), (200, 1500, 6)])
def test_a_last_round_of_cut_blocks(t, rows, columns, rest):
    """Blocks of 256 x 256 in rounds of 256, those of the last one whole, in halves or in quarters; of all three products in turn."""
    assert -(-rows // 256) * -(-columns // 256) % 256 == rest
    with cc.option(cc.Option.real_block, 7):
        for M, N, K in ((rows, columns, 72), (rows, 37, columns), (100, rows, columns)):
            layer = run_layer(M, N, K, t, ACT.silu)
            assert all("cut" in layer.KernelName(product) for product in range(3))
        run_layer(70, 255, 577, t, ACT.gelu, pitches=(579, 581, 257), shift=1)


@pytest.mark.parametrize("K", [1, 7, 8, 9, 63, 64, 65, 127, 128, 129, 191, 200, 320, 333])
def test_every_length_of_the_sum_in_cut_blocks(K):
    with cc.option(cc.Option.real_block, 7):
        run_layer(260, 300, K, VT.bfloat16, ACT.none)
        run_layer(130, K, 520, VT.float16, ACT.none)


@pytest.mark.parametrize("K", [1, 8, 31, 32, 33, 64, 127, 128, 129, 160, 1000, 1023, 1024, 1025, 1056, 1152, 1999, 2048, 2080, 3100])
def test_every_length_of_the_sum_of_few_rows(K):
    """Whole steps of all waves, the whole 32 values behind them, and the end."""
    layer = run_layer(3, 20, K, VT.bfloat16, ACT.none)
    assert "linear_rows" in layer.KernelName()
    run_layer(3, 20, K, VT.float16, ACT.none, pitches=(K + 3, K + 1, 20), shift=1)


def test_two_layers_at_once():
    """On two streams, with parts of K joined and ends of rows copied in scratch memory of their own: the bits of one after the other."""
    M, N, K, t = 70, 129, 4099, VT.bfloat16
    gen = torch.Generator().manual_seed(8)
    layers, held = [], []
    for _ in range(2):
        side = torch.cuda.Stream()
        with cc.option(cc.Option.real_block, 3 + 256 * 4):
            layers.append((cc.FusedLinear(M, N, K, 0, side.cuda_stream, t, ACT.gelu), side))
        ins = [made(gen, r, c, t).to(HALF[t]).cuda() for r, c in ((M, K), (N, K), (M, N))]
        outs = [torch.zeros(s, dtype=d, device="cuda") for s, d in (((M, N), HALF[t]), ((M, N), HALF[t]), ((M, K), HALF[t]),
                                                                    ((N, K), torch.float32), ((N,), torch.float32))]
        held.append((ins, outs))

    def run(layer, both):
        (x, w, dy), (y, z, dx, dw, db) = both
        layer.Forward(x.data_ptr(), w.data_ptr(), 0, 0, y.data_ptr(), z.data_ptr())
        layer.Backward(dy.data_ptr(), z.data_ptr(), x.data_ptr(), w.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr())

    torch.cuda.synchronize()
    alone = []
    for (layer, _), both in zip(layers, held):
        run(layer, both)
        torch.cuda.synchronize()
        alone.append([v.clone() for v in both[1]])
    torch.cuda.synchronize()
    for _ in range(20):
        for (layer, _), both in zip(layers, held):
            run(layer, both)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for want, both in zip(alone, held) for a, b in zip(want, both[1]))
