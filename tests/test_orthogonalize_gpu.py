"""Orthogonalize against the iteration in 64 bits.

Tolerances, relative Frobenius error: that of the exact result rounded to the type, and for the chain of products: bfloat16,
rounded to 11 bits, 2.1e-4 of the norm a rounding: fifteen of them, which the iteration may stretch while it raises small
singular values (a factor of 3.44 a step, mostly early): 2e-3. float16 and float32, 22 bits: 1e-5, fifteen roundings of
2^-22 and sums whose length adds to them."""
import itertools

import pytest
import torch

import ccglib_amd as cc
from scaled_util import WIDE, orthogonalized, stream

pytestmark = pytest.mark.gpu
VT = cc.ValueType
CHAIN = {VT.bfloat16: 2e-3, VT.float16: 1e-5, VT.float32: 1e-5}


def update(B, M, N, t, gen, size=1e-3):
    k = max(1, min(M, N) // 8)
    low = torch.randn((B, M, k), generator=gen) @ torch.randn((B, k, N), generator=gen) / k ** 0.5
    return ((low + torch.randn((B, M, N), generator=gen)) * size).to(WIDE[t]).cuda()


def run(g, t, out=None, **more):
    B, M, N = g.shape
    out = torch.empty_like(g) if out is None else out
    op = cc.Orthogonalize(B, M, N, 0, stream(), t, **more)
    op.Run(g.data_ptr(), out.data_ptr())
    torch.cuda.synchronize()
    return out, op


def near(got, want, t):
    off = float((got.double().cpu() - want).norm() / want.norm())
    rounding = float((want.to(WIDE[t]).double() - want).norm() / want.norm())
    return off <= rounding + CHAIN[t]


SIZES = [(1, 1, 1), (2, 1, 7), (2, 7, 1), (3, 2, 3), (1, 16, 24), (2, 63, 65), (4, 128, 96), (1, 130, 500), (1, 500, 130), (1, 64, 4096),
         (1, 300, 301), (2, 577, 300), (40, 40, 72), (1, 1030, 700)]


@pytest.mark.parametrize("t", list(WIDE))
def test_sizes(t):
    gen = torch.Generator().manual_seed(1)
    for B, M, N in SIZES:
        g = update(B, M, N, t, gen)
        got, _ = run(g, t)
        assert near(got, orthogonalized(g), t), (B, M, N)


@pytest.mark.parametrize("t", list(WIDE))
@pytest.mark.parametrize("shape,parts", [(1, 1), (1, 3), (2, 1), (2, 2), (3, 1), (3, 5)])
def test_every_block_shape(t, shape, parts):
    """The shapes that the sizes would not choose, K in one part and in several."""
    gen = torch.Generator().manual_seed(10)
    for B, M, N in [(2, 5, 9), (1, 70, 260), (2, 280, 130), (1, 400, 330)]:
        g = update(B, M, N, t, gen)
        with cc.option(cc.Option.real_block, shape + 256 * parts):
            got, _ = run(g, t)
        assert near(got, orthogonalized(g), t), (B, M, N)


@pytest.mark.parametrize("t", list(WIDE))
@pytest.mark.parametrize("M,N", [(2100, 2300), (3000, 520), (520, 3000)])
def test_large_blocks(t, M, N):
    g = update(1, M, N, t, torch.Generator().manual_seed(2))
    got, _ = run(g, t)
    want = g.double()[0] / (g.double()[0].norm() + 1e-7)
    for _ in range(5):
        s = want @ want.t().contiguous() if M <= N else want.t().contiguous() @ want
        p = -4.7750 * s + 2.0315 * (s @ s)
        want = 3.4445 * want + (p @ want if M <= N else want @ p)
    assert near(got, want.cpu()[None], t)


@pytest.mark.parametrize("t", list(WIDE))
@pytest.mark.parametrize("steps,coefficients", [(1, (3.4445, -4.7750, 2.0315)), (2, (1.5, -0.5, 0.0)), (9, (2.0, -1.5, 0.5))])
def test_other_iterations(t, steps, coefficients):
    gen = torch.Generator().manual_seed(3)
    for M, N in [(60, 100), (200, 130)]:
        g = update(2, M, N, t, gen)
        got, _ = run(g, t, steps=steps, coefficients=coefficients)
        assert near(got, orthogonalized(g, steps, coefficients), t)


@pytest.mark.parametrize("t", list(WIDE))
def test_singular_values(t):
    """What it is for: with the default steps the singular values of a well-conditioned update end between 0.6 and 1.3."""
    g = torch.randn((1, 100, 300), generator=torch.Generator().manual_seed(4)).to(WIDE[t]).cuda()
    got, _ = run(g, t)
    s = torch.linalg.svdvals(got[0].double().cpu())
    assert 0.6 < float(s.min()) and float(s.max()) < 1.3


@pytest.mark.parametrize("t", list(WIDE))
@pytest.mark.parametrize("size", [3e4, 1.0, 6e-5])
def test_any_size_of_values(t, size):
    gen = torch.Generator().manual_seed(5)
    for M, N in [(70, 90), (200, 190)]:
        g = update(1, M, N, t, gen, size=size if t != VT.float16 else min(size, 1e3))
        got, _ = run(g, t, epsilon=0.0)
        assert near(got, orthogonalized(g, epsilon=0.0), t)


@pytest.mark.parametrize("t", [VT.bfloat16, VT.float32])
@pytest.mark.parametrize("exponent", [-100, -60, 60, 100])
def test_values_whose_squares_leave_32_bits(t, exponent):
    gen = torch.Generator().manual_seed(6)
    for M, N in [(70, 90), (200, 190)]:
        g = update(1, M, N, t, gen, size=1.0)
        want = orthogonalized(g, epsilon=0.0)
        got, _ = run((g.double() * 2.0 ** exponent).to(WIDE[t]), t, epsilon=0.0)
        assert near(got, want, t)


@pytest.mark.parametrize("t", list(WIDE))
def test_zeros_and_what_is_no_number(t):
    """A matrix of zeros stays one; a NaN or an infinity makes its own matrix NaN, and no other."""
    gen = torch.Generator().manual_seed(7)
    for M, N in [(40, 60), (150, 140)]:
        g = update(5, M, N, t, gen)
        g[1] = 0
        g[2, 3, 4] = float("nan")
        g[3, M - 1, N - 1] = float("-inf")
        got, _ = run(g, t)
        assert not got[1].any()
        assert bool(torch.isnan(got[2]).all()) and bool(torch.isnan(got[3]).all())
        rest = [0, 4]
        assert near(got[rest], orthogonalized(g[rest]), t)


@pytest.mark.parametrize("t", list(WIDE))
@pytest.mark.parametrize("M,N", [(40, 60), (60, 40), (260, 131)])
def test_in_place_and_rows_apart(t, M, N):
    gen = torch.Generator().manual_seed(8)
    g = update(2, M, N, t, gen)
    want, _ = run(g, t)
    same = g.clone()
    run(same, t, out=same)
    assert torch.equal(same, want)
    pitch_in, pitch_out = N + 5, N + 3
    apart = torch.zeros((2, M, pitch_in), dtype=WIDE[t], device="cuda")
    apart[:, :, :N] = g
    out = torch.full((2, M, pitch_out), 7.0, dtype=WIDE[t], device="cuda")
    cc.Orthogonalize(2, M, N, 0, stream(), t, input_pitch=pitch_in, output_pitch=pitch_out).Run(apart.data_ptr(), out.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(out[:, :, :N], want) and bool((out[:, :, N:] == 7).all())


@pytest.mark.parametrize("t", [VT.bfloat16, VT.float32])
@pytest.mark.parametrize("B,M,N", [(3, 100, 80), (1, 700, 2000)])
def test_same_bits_again_in_a_graph_and_on_another_stream(t, B, M, N):
    gen = torch.Generator().manual_seed(9)
    g, other = update(B, M, N, t, gen), update(B, M, N, t, gen)
    want, _ = run(g, t)
    want_other, _ = run(other, t)
    side = torch.cuda.Stream()
    op = cc.Orthogonalize(B, M, N, 0, side.cuda_stream, t)
    buffer, out = g.clone(), torch.zeros_like(g)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        op.Run(buffer.data_ptr(), out.data_ptr())
    for k in range(4):
        buffer.copy_(g if k % 2 else other)
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want if k % 2 else want_other)
        out.zero_()
        torch.cuda.synchronize()
        op.Run(buffer.data_ptr(), out.data_ptr())
        torch.cuda.synchronize()
        assert torch.equal(out, want if k % 2 else want_other)


def test_empty_and_refusals_at_run():
    for B, M, N in [(0, 4, 4), (1, 0, 4), (1, 4, 0)]:
        cc.Orthogonalize(B, M, N, 0, stream()).Run(0, 0)
    t = torch.zeros(256, device="cuda")
    op = cc.Orthogonalize(1, 4, 4, 0, stream(), VT.float32)
    with pytest.raises(RuntimeError, match="null pointer"):
        op.Run(0, t.data_ptr())
    with pytest.raises(RuntimeError, match="null pointer"):
        op.Run(t.data_ptr(), 0)
    with pytest.raises(RuntimeError, match="misaligned"):
        op.Run(t.data_ptr() + 2, t.data_ptr())


@pytest.mark.parametrize("parts", [1, 3])
def test_blocks_of_eight_waves(parts):
    gen = torch.Generator().manual_seed(11)
    t = VT.bfloat16
    for B, M, N in [(2, 5, 9), (1, 70, 260), (2, 280, 130), (1, 400, 330)]:
        g = update(B, M, N, t, gen)
        with cc.option(cc.Option.real_block, 4 + 256 * parts):
            got, _ = run(g, t)
        assert near(got, orthogonalized(g), t), (B, M, N)


def test_as_many_blocks_as_units():
    t = VT.bfloat16
    g = update(1, 1000, 4000, t, torch.Generator().manual_seed(12))
    got, _ = run(g, t)
    assert near(got, orthogonalized(g), t)


@pytest.mark.parametrize("M,N", [(64, 128), (600, 700), (1000, 1000)])
@pytest.mark.parametrize("seed", [3, 4, 5])
def test_no_row_of_a_32_bit_update_is_worse_than_its_roundings(M, N, seed):
    """Every value of the chain has 22 bits, three matrices a step, five steps: 15 x 2^-22 = 3.6e-6 of a row. A value whose two
    parts do not belong together is 2^-11 of itself off, 1.5e-5 and more of its row."""
    g = torch.randn((2, M, N), generator=torch.Generator().manual_seed(seed)).cuda()
    got, _ = run(g, VT.float32)
    want = orthogonalized(g)
    off = (got.double().cpu() - want).norm(dim=2) / want.norm(dim=2)
    assert float(off.max()) < 4e-6


@pytest.mark.parametrize("parts", [1, 3])
def test_blocks_of_192(parts):
    gen = torch.Generator().manual_seed(13)
    t = VT.bfloat16
    for B, M, N in [(2, 5, 9), (1, 70, 260), (2, 280, 130), (1, 400, 330), (1, 390, 500)]:
        g = update(B, M, N, t, gen)
        with cc.option(cc.Option.real_block, 5 + 256 * parts):
            got, _ = run(g, t)
        assert near(got, orthogonalized(g), t), (B, M, N)


@pytest.mark.parametrize("t", list(WIDE))
@pytest.mark.parametrize("M,N", [(333, 301), (150, 517), (60, 100)])
def test_a_matrix_of_nan_leaves_nothing_behind(t, M, N):
    """The object's next run, with an ordinary matrix, is that of a new object."""
    gen = torch.Generator().manual_seed(14)
    g = update(2, M, N, t, gen)
    want, _ = run(g, t)
    bad, out = torch.full_like(g, float("nan")), torch.empty_like(g)
    op = cc.Orthogonalize(2, M, N, 0, stream(), t)
    for x in (bad, g):
        op.Run(x.data_ptr(), out.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(out, want)
