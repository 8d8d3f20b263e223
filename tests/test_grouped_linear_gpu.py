"""GroupedLinear: y, z, dx, dW and dbias of every expert against 64 bits (bounds: linear_util.py), for offsets that leave experts
without rows, rows without an expert, and all rows to one; what belongs to no expert is neither read nor written."""
import itertools
import math

import pytest
import torch

import ccglib_amd as cc
from linear_util import ACT, HALF, TORCH, VT, among_nan, backward, check, forward, stream

pytestmark = pytest.mark.gpu

SPANS = {
    "even": lambda M, E: [round(e * M / E) for e in range(E + 1)],
    "none of most": lambda M, E: [0] * (E // 2 + 1) + [M] * (E - E // 2),
    "all of the last": lambda M, E: [0] * E + [M],
    "rows before and behind": lambda M, E: [min(M, 3 + e * max(0, M - 8) // E) for e in range(E + 1)],
    "no rows": lambda M, E: [0] * (E + 1),
    "one each": lambda M, E: [min(e, M) for e in range(E + 1)],
}


def run_layer(E, M, N, K, t, activation, offsets, gradient_type=VT.float32, pitches=(0, 0, 0), shift=0, accumulate=False, held=None):
    """One forward and one backward pass, both checked. held: what the device's offsets say, where that differs from what counts."""
    gen = torch.Generator().manual_seed(E + M + 7 * N + 11 * K)
    xp, wp, yp = pitches

    def normal(rows, columns, scale=1.0):
        return (torch.randn((rows, columns), generator=gen, dtype=torch.float64) * scale).to(HALF[t])
    x, w, b, dy = normal(M, K), normal(E * N, K, max(1, K) ** -0.5), normal(E, N), normal(M, N, 0.1)
    mine = torch.zeros(M, dtype=torch.bool)
    mine[offsets[0]:offsets[E]] = True
    x[~mine], dy[~mine] = math.nan, math.nan            # (rows of no expert: not read)
    dev = {"x": among_nan(x, xp, shift), "w": among_nan(w, wp, shift), "b": among_nan(b), "dy": among_nan(dy, yp, shift)}
    o = torch.tensor(held or offsets, dtype=torch.int32, device="cuda")
    marks = [among_nan(torch.full(s, 77.0, dtype=HALF[t]), p, shift) for s, p in (((M, N), yp), ((M, N), yp), ((M, K), xp))]
    y, z, dx = marks
    layer = cc.GroupedLinear(E, M, N, K, 0, stream(), t, activation, gradient_type, True, xp, wp, yp)
    layer.Forward(dev["x"].data_ptr(), o.data_ptr(), dev["w"].data_ptr(), dev["b"].data_ptr(), 0, y.data_ptr(), z.data_ptr())
    torch.cuda.synchronize()
    old_w, old_b = normal(E * N, K), normal(E, N)
    dw, db = among_nan(old_w.to(TORCH[gradient_type]), wp, shift), among_nan(old_b.to(TORCH[gradient_type]))
    layer.Backward(dev["dy"].data_ptr(), z.data_ptr(), dev["x"].data_ptr(), o.data_ptr(), dev["w"].data_ptr(), dx.data_ptr(),
                   dw.data_ptr(), db.data_ptr(), accumulate=accumulate)
    torch.cuda.synchronize()
    for out in marks:
        assert bool((out[~mine.cuda()] == 77.0).all()), "rows of no expert"
    for e in range(E):
        rows, ws = slice(offsets[e], offsets[e + 1]), slice(e * N, (e + 1) * N)
        x64, w64, b64, dy64 = (v.double().cuda() for v in (x[rows], w[ws], b[e], dy[rows]))
        zw, yw, ez, ey = forward(x64, w64, b64, None, activation)
        check(z[rows], zw, ez, "z of %d" % e)
        check(y[rows], yw, ey, "y of %d" % e)
        (dxw, dww, dbw), (edx, edw, edb) = backward(dy64, z[rows].double(), x64, w64, activation, HALF[t])
        if accumulate:
            dww, dbw = dww + old_w[ws].cuda().double(), dbw + old_b[e].cuda().double()
            edw, edb = edw + 2.0 ** -23 * dww.abs(), edb + 2.0 ** -23 * dbw.abs()
        check(dx[rows], dxw, edx, "dx of %d" % e)
        check(dw[ws], dww, edw, "dw of %d" % e)
        check(db[e], dbw, edb, "db of %d" % e)
    return layer


@pytest.mark.parametrize("t,activation", [(VT.bfloat16, ACT.silu), (VT.float16, ACT.none)])
@pytest.mark.parametrize("spans", list(SPANS))
@pytest.mark.parametrize("E,M,N,K", [(1, 40, 30, 50), (4, 300, 130, 200), (5, 7, 64, 65), (70, 200, 40, 24), (130, 333, 17, 9)])
def test_forward_and_backward(t, activation, spans, E, M, N, K):
    run_layer(E, M, N, K, t, activation, SPANS[spans](M, E))


@pytest.mark.parametrize("shape", range(1, 7))
@pytest.mark.parametrize("spans", ["even", "rows before and behind", "one each"])
def test_every_shape(shape, spans):
    with cc.option(cc.Option.real_block, shape):
        run_layer(3, 700, 265, 330, VT.bfloat16, ACT.gelu, SPANS[spans](700, 3))
        run_layer(9, 100, 24, 136, VT.float16, ACT.relu, SPANS[spans](100, 9))


@pytest.mark.parametrize("shape", range(0, 7))
@pytest.mark.parametrize("pitches,shift", [((584, 584, 264), 0), ((577, 577, 255), 3), ((579, 581, 257), 1)])
def test_distances_and_addresses(shape, pitches, shift):
    with cc.option(cc.Option.real_block, shape):
        run_layer(3, 70, 255, 577, VT.bfloat16, ACT.gelu, [0, 30, 31, 70], pitches=pitches, shift=shift)
        run_layer(3, 9, 3, 5, VT.float16, ACT.none, [0, 2, 8, 9], pitches=(5, 6, 7), shift=shift)
        run_layer(2, 90, 1, 1, VT.float16, ACT.relu, [0, 88, 90], pitches=(1, 1, 1), shift=shift)


@pytest.mark.parametrize("gradient_type,accumulate", [(VT.float32, True), (VT.bfloat16, False)])
def test_gradients_of_weights_in_either_type(gradient_type, accumulate):
    run_layer(3, 130, 70, 90, VT.bfloat16, ACT.none, [0, 60, 60, 130], gradient_type, accumulate=accumulate)


@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65, 127, 128, 129, 191, 200, 255, 257])
def test_every_length_of_an_experts_rows(rows):
    M = 2 * rows + 3
    for shape in range(1, 7):
        with cc.option(cc.Option.real_block, shape):
            run_layer(3, M, 40, 24, VT.bfloat16, ACT.none, [0, rows, rows + 3, M])


@pytest.mark.parametrize("spans", list(SPANS))
@pytest.mark.parametrize("E,M,N,K", [(1, 2, 33, 1031), (40, 60, 17, 1030), (66, 100, 40, 24), (100, 3, 50, 2048)])
def test_few_rows(spans, E, M, N, K):
    """What the kernel for a few rows takes: an expert may have more than 16 of them."""
    layer = run_layer(E, M, N, K, VT.bfloat16, ACT.silu, SPANS[spans](M, E), pitches=(K + 1, K, N), shift=E % 2)
    assert "linear_rows" in layer.KernelName()


def test_offsets_outside_the_rows_count_as_the_nearer_end():
    run_layer(4, 50, 24, 40, VT.bfloat16, ACT.none, [0, 10, 50, 50, 50], held=[-7, 10, 51, 2 ** 31 - 1, 60])


@pytest.mark.parametrize("M,N,K", [(0, 5, 6), (5, 0, 6), (5, 6, 0)])
def test_empty_extents(M, N, K):
    run_layer(2, M, N, K, VT.bfloat16, ACT.gelu, [0, M // 2, M])


def test_one_expert_is_a_fused_layer():
    """The same kernels at the same sizes: the same bits."""
    M, N, K, t = 190, 300, 264, VT.bfloat16
    gen = torch.Generator().manual_seed(2)
    x, w, z, dy = (torch.randn(s, generator=gen).to(HALF[t]).cuda() for s in ((M, K), (N, K), (M, N), (M, N)))
    o = torch.tensor([0, M], dtype=torch.int32, device="cuda")
    got = []
    with cc.option(cc.Option.real_block, 2 + 256):       # (one part of K, as grouped products have)
        fused = cc.FusedLinear(M, N, K, 0, stream(), t, ACT.silu)
        grouped = cc.GroupedLinear(1, M, N, K, 0, stream(), t, ACT.silu)
    for layer, more in ((fused, ()), (grouped, (o.data_ptr(),))):
        y, dx, dw, db = torch.empty_like(z), torch.empty_like(x), torch.empty((N, K), device="cuda"), torch.empty(N, device="cuda")
        layer.Forward(x.data_ptr(), *more, w.data_ptr(), 0, 0, y.data_ptr())
        layer.Backward(dy.data_ptr(), z.data_ptr(), x.data_ptr(), *more, w.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr())
        torch.cuda.synchronize()
        got.append((y, dx, dw, db))
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_refusals_of_a_run():
    t = torch.zeros(4096, dtype=torch.bfloat16, device="cuda")
    p = t.data_ptr()
    layer = cc.GroupedLinear(2, 4, 4, 4, 0, stream(), activation=ACT.gelu, gradient_type=VT.bfloat16)
    with pytest.raises(RuntimeError, match="null pointer: GroupedLinear, offsets"):
        layer.Forward(p, 0, p, 0, 0, p)
    with pytest.raises(RuntimeError, match="misaligned offsets"):
        layer.Forward(p, p + 2, p, 0, 0, p)
    with pytest.raises(RuntimeError, match="null pointer: GroupedLinear, offsets"):
        layer.Backward(p, p, p, 0, p, p, p)
    with pytest.raises(RuntimeError, match="null pointer: GroupedLinear, z"):
        layer.Backward(p, 0, p, p, p, p, p)
    with pytest.raises(RuntimeError, match="added to are float32"):
        layer.Backward(p, p, p, p, p, p, p, accumulate=True)
    with pytest.raises(RuntimeError, match="without training"):
        cc.GroupedLinear(2, 4, 4, 4, 0, stream(), training=False).Backward(p, p, p, p, p, p, p)


@pytest.mark.parametrize("M,K", [(600, 72), (11, 1030)])
def test_operands_beyond_32_bits(M, K):
    """Rows 8 MiB apart: 5 GB of W, which experts lie all over."""
    run_layer(4, M, 150, K, VT.float16, ACT.silu, [0, 3, 5, 9, M], pitches=(1 << 22,) * 3)


@pytest.mark.parametrize("spans", list(SPANS))
@pytest.mark.parametrize("M,N,K", [(4000, 5100, 72), (3900, 40, 6100), (300, 520, 200)])
def test_a_last_round_of_cut_blocks(spans, M, N, K):
    """How many blocks there are is known to the kernel alone."""
    with cc.option(cc.Option.real_block, 7):
        layer = run_layer(3, M, N, K, VT.bfloat16, ACT.silu, SPANS[spans](M, 3))
        assert ["cut" in layer.KernelName(product) for product in range(3)] == [True, True, False]
        run_layer(3, 70, 255, 577, VT.float16, ACT.gelu, [0, 30, 31, 70], pitches=(579, 581, 257), shift=1)


@pytest.mark.parametrize("gradient_type", [VT.float32, VT.bfloat16])
@pytest.mark.parametrize("E", [1, 7, 64, 65])
def test_experts_of_very_different_loads(E, gradient_type):
    """dW's experts take turns in classes of their rows' number: each of them once, whatever the numbers are."""
    counts = [(700 if e % 9 == 4 else 130 if e % 5 == 2 else e % 3 * 20) for e in range(E)]
    offsets = [3 + sum(counts[:e]) for e in range(E + 1)]
    for shape in (1, 2, 4):
        with cc.option(cc.Option.real_block, shape):
            run_layer(E, offsets[-1] + 5, 70, 330, VT.bfloat16, ACT.none, offsets, gradient_type, accumulate=gradient_type == VT.float32)


@pytest.mark.parametrize("shape", [2, 7])
def test_two_graphs_of_one_layer_with_changing_loads(shape):
    """They share its scratch memory and are replayed in turn; each replay takes the offsets that it finds, and gives the bits of an eager
    run of another object."""
    E, M, N, K, t = 5, 700, 264, 330, VT.bfloat16
    gen = torch.Generator().manual_seed(shape)
    side = torch.cuda.Stream()
    with cc.option(cc.Option.real_block, shape):
        shared = cc.GroupedLinear(E, M, N, K, 0, side.cuda_stream, t, ACT.gelu)
        other = cc.GroupedLinear(E, M, N, K, 0, stream(), t, ACT.gelu)

    def buffers():
        ins = [torch.randn(s, generator=gen).to(HALF[t]).cuda() for s in ((M, K), (E * N, K), (M, N))]
        outs = [torch.zeros(s, dtype=d, device="cuda") for s, d in (((M, N), HALF[t]), ((M, N), HALF[t]), ((M, K), HALF[t]),
                                                                    ((E * N, K), torch.float32), ((E, N), torch.float32))]
        return ins, outs, torch.zeros(E + 1, dtype=torch.int32, device="cuda")

    def run(layer, held):
        (x, w, dy), (y, z, dx, dw, db), o = held
        layer.Forward(x.data_ptr(), o.data_ptr(), w.data_ptr(), 0, 0, y.data_ptr(), z.data_ptr())
        layer.Backward(dy.data_ptr(), z.data_ptr(), x.data_ptr(), o.data_ptr(), w.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr())

    sets, graphs = [buffers(), buffers()], []
    torch.cuda.synchronize()
    for held in sets:
        with torch.cuda.stream(side):
            run(shared, held)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            run(shared, held)
        graphs.append(graph)
    for spans in list(SPANS.values())[:4]:
        for held, graph in zip(sets, graphs):
            held[2].copy_(torch.tensor(spans(M, E), dtype=torch.int32))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            again = (held[0], [torch.zeros_like(v) for v in held[1]], held[2])
            run(other, again)
            torch.cuda.synchronize()
            first, until = int(held[2][0]), int(held[2][-1])
            for got, want in zip(held[1][:3], again[1][:3]):
                assert torch.equal(got[first:until], want[first:until])
            assert all(torch.equal(got, want) for got, want in zip(held[1][3:], again[1][3:]))


@pytest.mark.parametrize("shape", [0, 1, 2, 7])
def test_offsets_that_fall_harm_nothing_else(shape):
    """Results are unspecified; what lies around the outputs is left alone."""
    E, M, N, K, t = 4, 300, 70, 90, VT.bfloat16
    gen = torch.Generator().manual_seed(4)
    x, w, dy = (among_nan(torch.randn(s, generator=gen).to(HALF[t])) for s in ((M, K), (E * N, K), (M, N)))
    outs = [among_nan(torch.zeros(s, dtype=d)) for s, d in (((M, N), HALF[t]), ((M, N), HALF[t]), ((M, K), HALF[t]),
                                                            ((E * N, K), torch.float32), ((E, N), torch.float32))]
    with cc.option(cc.Option.real_block, shape):
        layer = cc.GroupedLinear(E, M, N, K, 0, stream(), t, ACT.silu)
    y, z, dx, dw, db = outs
    for offsets in ([0, 300, 0, 300, 0], [300, 200, 100, 50, 0], [-5, 2 ** 31 - 1, -2 ** 31, 299, 3]):
        o = torch.tensor(offsets, dtype=torch.int32, device="cuda")
        layer.Forward(x.data_ptr(), o.data_ptr(), w.data_ptr(), 0, 0, y.data_ptr(), z.data_ptr())
        layer.Backward(dy.data_ptr(), z.data_ptr(), x.data_ptr(), o.data_ptr(), w.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr())
        torch.cuda.synchronize()
    for out in outs:
        size = out.numel()
        whole = torch.empty(0, dtype=out.dtype, device="cuda").set_(out.untyped_storage())
        at = out.storage_offset()
        assert bool(whole[:at].isnan().all()) and bool(whole[at + size:].isnan().all())
