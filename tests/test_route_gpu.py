"""Route and Combine against plain statements in 64 bits: choices, places and offsets exactly, weights, sums and gradients within
the roundings of 32 bits; ties, masked and missing experts, NaN, one tile of tokens and many, rows that no slot names, slots that
are no rows; and the two together with GroupedLinear as a layer of experts, captured and replayed."""
import itertools
import math

import pytest
import torch

import ccglib_amd as cc
from linear_util import ACT, HALF, TORCH, VT, among_nan, check, routed, stream

pytestmark = pytest.mark.gpu


def run_route(logits, k, normalize, seed=0):
    T, E = logits.shape
    t = {v: n for n, v in TORCH.items()}[logits.dtype]
    d = logits.cuda()
    experts, slots = (torch.full((T, k), -1, dtype=torch.int32, device="cuda") for _ in range(2))
    weights, offsets = torch.full((T, k), math.nan, device="cuda"), torch.full((E + 1,), -1, dtype=torch.int32, device="cuda")
    route = cc.Route(T, E, k, 0, stream(), t, normalize)
    route.Run(d.data_ptr(), experts.data_ptr(), weights.data_ptr(), offsets.data_ptr(), slots.data_ptr())
    dweights = torch.randn((T, k), generator=torch.Generator().manual_seed(seed)).cuda()
    dlogits = torch.full((T, E), math.nan, dtype=logits.dtype, device="cuda")
    route.Backward(0 if normalize else d.data_ptr(), experts.data_ptr(), weights.data_ptr(), dweights.data_ptr(), dlogits.data_ptr())
    torch.cuda.synchronize()
    return experts.cpu(), weights.cpu(), offsets.cpu(), slots.cpu(), dweights.cpu(), dlogits.cpu()


def check_route(logits, k, normalize):
    T, E = logits.shape
    experts, weights, offsets, slots, dweights, dlogits = run_route(logits, k, normalize)
    e, w, o, s = routed(logits, k, normalize)
    assert torch.equal(experts.long(), e) and offsets.tolist() == o and torch.equal(slots.long(), s)
    # exp(l - top) is |l - top| + 4 steps of 2^-23 off (at most 88 where it is not 0), sums E more, the quotient one
    error = (88 + 8 + E) * 2.0 ** -23
    check(weights, w, error * w + 1e-37, "weights")
    dw = dweights.double()
    inner = (w * dw).sum(dim=1, keepdim=True)
    size = (w * dw.abs()).sum(dim=1, keepdim=True)
    full = torch.zeros((T, E), dtype=torch.float64).scatter_(1, e, dw)
    if normalize:
        p = torch.zeros((T, E), dtype=torch.float64).scatter_(1, e, w)
    else:
        top = logits.double().amax(dim=1, keepdim=True)
        p = torch.exp(logits.double() - torch.where(top == -math.inf, torch.zeros_like(top), top))
        p = torch.where(p.sum(dim=1, keepdim=True) == 0, torch.zeros_like(p), p / p.sum(dim=1, keepdim=True))
    check(dlogits, p * (full - inner), 3 * error * p * (full.abs() + size) + 1e-37, "dlogits")


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("t", list(TORCH))
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 8), (3, 16, 16), (64, 17, 4), (65, 64, 2), (100, 100, 7), (200, 128, 8),
                                   (70, 255, 3), (66, 256, 16), (90, 257, 5), (40, 512, 9), (33, 1000, 2), (65, 1024, 16)])
def test_route(t, T, E, k, normalize):
    gen = torch.Generator().manual_seed(T + E + k)
    check_route((torch.randn((T, E), generator=gen) * 3).to(TORCH[t]), k, normalize)


@pytest.mark.parametrize("T,E,k", [(16384, 8, 2), (16385, 24, 1), (20000, 130, 3), (40000, 3, 3)])
def test_many_tiles(T, E, k):
    gen = torch.Generator().manual_seed(T)
    check_route((torch.randn((T, E), generator=gen) + torch.linspace(0, 3, E)).to(torch.bfloat16), k, False)


def test_ties_go_to_the_lower_number_and_zeros_are_alike():
    logits = torch.tensor([[0.0, -0.0, 0.0, 1.0], [-0.0, 0.0, -0.0, -1.0], [2.0, 2.0, 2.0, 2.0], [-math.inf] * 4])
    for k in (1, 2, 3, 4):
        check_route(logits, k, True)
        check_route(logits.half(), k, False)


@pytest.mark.parametrize("normalize", [True, False])
def test_masked_experts(normalize):
    """Experts at -inf, or at the lowest number of the type, are chosen last and weigh nothing; where all of them are masked, all
    weigh nothing (-inf) or the same (the lowest number)."""
    gen = torch.Generator().manual_seed(1)
    logits = torch.randn((40, 30), generator=gen)
    logits[:, 5:25] = -math.inf
    logits[3] = -math.inf
    logits[4, 1:] = -math.inf
    logits[6] = torch.finfo(torch.float32).min
    logits[7, 2:] = torch.finfo(torch.float32).min
    check_route(logits, 12, normalize)


def test_logits_that_are_not_finite_choose_experts_all_the_same():
    logits = torch.zeros((4, 20))
    logits[0, 7], logits[0, 3] = math.nan, math.inf
    logits[1] = math.nan
    logits[2, 11] = math.inf
    experts, weights, offsets, slots, _, _ = run_route(logits, 3, True)
    assert experts[0].tolist() == [7, 3, 0] and experts[1].tolist() == [0, 1, 2] and experts[2].tolist() == [11, 0, 1]
    assert experts[3].tolist() == [0, 1, 2] and bool(weights[:3].isnan().any(dim=1).all()) and not bool(weights[3].isnan().any())
    assert sorted(slots.flatten().tolist()) == list(range(12)) and int(offsets[-1]) == 12


def test_no_tokens():
    offsets = torch.full((6,), -1, dtype=torch.int32, device="cuda")
    cc.Route(0, 5, 2, 0, stream()).Run(0, 0, 0, offsets.data_ptr(), 0)
    torch.cuda.synchronize()
    assert offsets.tolist() == [0] * 6


def run_combine(T, k, N, t, rows, weighted, y_pitch=0, out_pitch=0, shift=0, holes=False):
    gen = torch.Generator().manual_seed(T + k + N)

    def normal(r, c):
        return torch.randn((r, c), generator=gen).to(HALF[t])
    y, x, dout = normal(rows, N), normal(T, N), normal(T, N)
    slots = torch.randperm(rows, generator=gen)[:T * k].reshape(T, k).to(torch.int32)
    if holes:
        slots[::3, 0], slots[1::4, k - 1], slots[2::5, k // 2] = -1, rows, 2 ** 31 - 1
    w = torch.rand((T, k), generator=gen) + 0.1
    d = {"y": among_nan(y, y_pitch, shift), "x": among_nan(x, out_pitch, shift), "dout": among_nan(dout, out_pitch, shift)}
    out = among_nan(torch.full((T, N), math.nan, dtype=HALF[t]), out_pitch, shift)
    spread, dy = (among_nan(torch.full((rows, N), 77.0, dtype=HALF[t]), y_pitch, shift) for _ in range(2))
    sd, wd, dw = slots.cuda(), w.cuda(), torch.full((T, k), math.nan, device="cuda")
    weights = wd.data_ptr() if weighted else 0
    combine = cc.Combine(T, k, N, 0, stream(), t, rows, y_pitch, out_pitch)
    combine.Run(d["y"].data_ptr(), sd.data_ptr(), weights, out.data_ptr())
    combine.Spread(d["x"].data_ptr(), sd.data_ptr(), weights, spread.data_ptr())
    combine.Backward(d["dout"].data_ptr(), d["y"].data_ptr(), sd.data_ptr(), weights, dy.data_ptr(), dw.data_ptr())
    torch.cuda.synchronize()
    w64 = w.double() if weighted else torch.ones((T, k), dtype=torch.float64)
    inside = (slots >= 0) & (slots < rows)
    at = torch.where(inside, slots, torch.zeros_like(slots)).long()
    picked = y.double()[at] * inside[:, :, None]                                   # [T][k][N]
    check(out, (w64[:, :, None] * picked).sum(dim=1), (k + 1) * 2.0 ** -23 * (w64[:, :, None] * picked.abs()).sum(dim=1), "out")
    check(dw, (picked * dout.double()[:, None]).sum(dim=2), (N + 1) * 2.0 ** -23 * (picked * dout.double()[:, None]).abs().sum(dim=2), "dweights")
    for got, source in ((spread, x), (dy, dout)):
        want, size = torch.full((rows, N), 77.0, dtype=torch.float64), torch.zeros((rows, N), dtype=torch.float64)
        value = w64[:, :, None] * source.double()[:, None]
        want[at[inside]], size[at[inside]] = value[inside], value[inside].abs()
        check(got, want, 2.0 ** -24 * size, "spread")
        unnamed = torch.ones(rows, dtype=torch.bool)
        unnamed[at[inside]] = False
        assert bool((got.cpu()[unnamed] == 77.0).all())
    # either gradient alone
    dy2, dw2 = torch.empty_like(dy), torch.empty_like(dw)
    dy2.copy_(dy)
    combine.Backward(d["dout"].data_ptr(), 0, sd.data_ptr(), weights, dy2.data_ptr() if not y_pitch else 0, 0)
    combine.Backward(d["dout"].data_ptr(), d["y"].data_ptr(), sd.data_ptr(), weights, 0, dw2.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(dy2, dy) and torch.equal(dw2, dw)


@pytest.mark.parametrize("t", list(HALF))
@pytest.mark.parametrize("T,k,N", [(1, 1, 1), (5, 2, 7), (33, 3, 100), (20, 8, 512), (9, 16, 513), (7, 5, 4096), (3, 2, 8195)])
def test_combine(t, T, k, N):
    run_combine(T, k, N, t, T * k, True)
    run_combine(T, k, N, t, T * k + 13, False, holes=k > 1)


@pytest.mark.parametrize("y_pitch,out_pitch,shift", [(104, 112, 0), (101, 103, 1), (130, 100, 5)])
def test_combine_at_distances(y_pitch, out_pitch, shift):
    run_combine(20, 4, 100, VT.bfloat16, 90, True, y_pitch, out_pitch, shift, holes=True)


def test_combine_of_nothing():
    w = torch.full((3, 2), math.nan, device="cuda")
    s = torch.zeros((3, 2), dtype=torch.int32, device="cuda")
    cc.Combine(3, 2, 0, 0, stream()).Backward(0, 0, s.data_ptr(), 0, 0, w.data_ptr())
    cc.Combine(0, 2, 8, 0, stream()).Run(0, 0, 0, 0)
    torch.cuda.synchronize()
    assert bool((w == 0).all())


def test_refusals_of_a_run():
    t = torch.zeros(4096, device="cuda")
    p = t.data_ptr()
    route = cc.Route(4, 8, 2, 0, stream())
    for i, name in enumerate(("logits", "experts", "weights", "offsets", "slots")):
        args = [p] * 5
        args[i] = 0
        with pytest.raises(RuntimeError, match="null pointer: Route, " + name):
            route.Run(*args)
        args[i] = p + 2
        with pytest.raises(RuntimeError, match="misaligned " + name):
            route.Run(*args)
    with pytest.raises(RuntimeError, match="null pointer: Route, logits"):
        cc.Route(4, 8, 2, 0, stream(), normalize=False).Backward(0, p, p, p, p)
    combine = cc.Combine(4, 2, 8, 0, stream())
    for i, name in enumerate(("y", "slots", None, "output")):
        args = [p] * 4
        if name:
            args[i] = 0
            with pytest.raises(RuntimeError, match="null pointer: Combine, " + name):
                combine.Run(*args)
        args[i] = p + 1
        with pytest.raises(RuntimeError, match="misaligned"):
            combine.Run(*args)
    with pytest.raises(RuntimeError, match="null pointer: Combine, y"):
        combine.Backward(p, 0, p, p, p, p)


class ExpertLayer:
    """Route, rows to their experts, two grouped layers, and back; forward and backward."""

    def __init__(self, T, E, k, width, hidden, on, t=VT.bfloat16):
        rows = T * k
        self.route, self.combine = cc.Route(T, E, k, 0, on), cc.Combine(T, k, width, 0, on, t)
        self.up = cc.GroupedLinear(E, rows, hidden, width, 0, on, t, ACT.silu)
        self.down = cc.GroupedLinear(E, rows, width, hidden, 0, on, t)

        def half(*s):
            return torch.zeros(s, dtype=HALF[t], device="cuda")
        self.experts, self.slots = (torch.zeros((T, k), dtype=torch.int32, device="cuda") for _ in range(2))
        self.offsets = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
        self.weights, self.dweights, self.dlogits = (torch.zeros(s, device="cuda") for s in ((T, k), (T, k), (T, E)))
        self.xs, self.dxs, self.ys, self.dys = (half(rows, width) for _ in range(4))
        self.h, self.z, self.dh = (half(rows, hidden) for _ in range(3))
        self.out, self.dx = half(T, width), half(T, width)
        self.dw1, self.dw2 = torch.zeros((E, hidden, width), device="cuda"), torch.zeros((E, width, hidden), device="cuda")

    def run(self, x, logits, w1, w2, dout):
        p = lambda v: v.data_ptr()     # noqa: E731
        self.route.Run(p(logits), p(self.experts), p(self.weights), p(self.offsets), p(self.slots))
        self.combine.Spread(p(x), p(self.slots), 0, p(self.xs))
        self.up.Forward(p(self.xs), p(self.offsets), p(w1), 0, 0, p(self.h), p(self.z))
        self.down.Forward(p(self.h), p(self.offsets), p(w2), 0, 0, p(self.ys))
        self.combine.Run(p(self.ys), p(self.slots), p(self.weights), p(self.out))
        self.combine.Backward(p(dout), p(self.ys), p(self.slots), p(self.weights), p(self.dys), p(self.dweights))
        self.down.Backward(p(self.dys), 0, p(self.h), p(self.offsets), p(w2), p(self.dh), p(self.dw2))
        self.up.Backward(p(self.dh), p(self.z), p(self.xs), p(self.offsets), p(w1), p(self.dxs), p(self.dw1))
        self.combine.Run(p(self.dxs), p(self.slots), 0, p(self.dx))
        self.route.Backward(p(logits), p(self.experts), p(self.weights), p(self.dweights), p(self.dlogits))

    def results(self):
        return [v.clone() for v in (self.out, self.dx, self.dlogits, self.dw1, self.dw2, self.offsets, self.slots)]


def expert_inputs(T, E, width, hidden, seed):
    gen = torch.Generator().manual_seed(seed)
    x, dout = (torch.randn((T, width), generator=gen).bfloat16().cuda() for _ in range(2))
    logits = torch.randn((T, E), generator=gen).cuda()
    w1 = (torch.randn((E, hidden, width), generator=gen) * width ** -0.5).bfloat16().cuda()
    w2 = (torch.randn((E, width, hidden), generator=gen) * hidden ** -0.5).bfloat16().cuda()
    return x, logits, w1, w2, dout


def test_a_layer_of_experts():
    """Forward and gradients of the whole against autograd in 64 bits. Each of the six roundings to 16 bits on the longest way
    (h, y; dy, dh, dz, dx of rows, dx) is 2^-8 of a value at most and independent of the others: together below 6 * 2^-9 of a result's
    norm (an error that is uniform in +-1/2 step has a third of its square)."""
    T, E, k, width, hidden = 100, 6, 2, 72, 136
    inputs = expert_inputs(T, E, width, hidden, 0)
    layer = ExpertLayer(T, E, k, width, hidden, stream())
    layer.run(*inputs)
    torch.cuda.synchronize()
    x, logits, w1, w2, dout = (v.double().cpu().requires_grad_(True) for v in inputs)
    experts = routed(logits.detach(), k, True)[0]
    weights = torch.softmax(logits.gather(1, experts), dim=1)
    out = torch.zeros((T, width), dtype=torch.float64)
    for j in range(k):
        z = torch.bmm(w1[experts[:, j]], x[:, :, None])
        out = out + weights[:, j:j + 1] * torch.bmm(w2[experts[:, j]], z * torch.sigmoid(z))[:, :, 0]
    (out * dout.detach()).sum().backward()
    for got, want in ((layer.out, out.detach()), (layer.dx, x.grad), (layer.dlogits, logits.grad), (layer.dw1, w1.grad), (layer.dw2, w2.grad)):
        got = got.double().cpu()
        assert float((got - want).norm()) <= 6 * 2.0 ** -9 * float(want.norm())


def test_a_captured_layer_of_experts():
    """Two layers captured into two graphs, replayed in turn with other inputs among the program's own work, on a stream of their
    own: each replay gives the bits of an eager run (a third object)."""
    T, E, k, width, hidden = 90, 5, 2, 64, 130
    side = torch.cuda.Stream()
    eager = ExpertLayer(T, E, k, width, hidden, stream())
    held, graphs, layers = [], [], []
    for g in range(2):
        layer = ExpertLayer(T, E, k, width, hidden, side.cuda_stream)
        buffers = expert_inputs(T, E, width, hidden, g)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            layer.run(*buffers)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            layer.run(*buffers)
        held.append(buffers)
        graphs.append(graph)
        layers.append(layer)
    for r in range(3):
        for g in range(2):
            inputs = expert_inputs(T, E, width, hidden, 10 * r + g)
            for to, new in zip(held[g], inputs):
                to.copy_(new)
            torch.cuda.synchronize()
            graphs[g].replay()
            torch.cuda.synchronize()
            eager.run(*inputs)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(layers[g].results(), eager.results()))


def test_a_captured_fused_layer():
    """With parts of K joined in the workspace, and ends of rows copied there."""
    M, N, K = 30, 65, 2051
    gen = torch.Generator().manual_seed(0)
    x, w, dy, z = (torch.randn(s, generator=gen).half().cuda() for s in ((M, K), (N, K), (M, N), (M, N)))
    y, dx, dw, db = torch.zeros_like(dy), torch.zeros_like(x), torch.zeros((N, K), device="cuda"), torch.zeros(N, device="cuda")
    side = torch.cuda.Stream()
    layer = cc.FusedLinear(M, N, K, 0, side.cuda_stream, VT.float16, ACT.gelu)

    def run():
        layer.Forward(x.data_ptr(), w.data_ptr(), 0, 0, y.data_ptr())
        layer.Backward(dy.data_ptr(), z.data_ptr(), x.data_ptr(), w.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr())
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        run()
    for r in range(3):
        for v in (x, w, dy, z):
            v.copy_(torch.randn(v.shape, generator=gen))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in (y, dx, dw, db)]
        with torch.cuda.stream(side):
            run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (y, dx, dw, db)))


def test_the_most_tokens():
    """2^24 - 1 rows of 300 logits, more of them than 32 bits count, in more tiles than otherwise, since 16 bits count a tile's rows of an
    expert. Logits are a row's permutation of 0 to 299, so that all answers are known: 37 e + t = 299 or 298 modulo 300, 37 * 73 = 1."""
    T, E, k = (1 << 24) - 1, 300, 2
    logits = torch.empty((T, E), dtype=torch.float16, device="cuda")
    rows, step = torch.arange(T, device="cuda"), 1 << 20
    for at in range(0, T, step):
        logits[at:at + step] = (rows[at:at + step, None].int() + 37 * torch.arange(E, device="cuda", dtype=torch.int32)) % E
    experts, slots = (torch.full((T, k), -1, dtype=torch.int32, device="cuda") for _ in range(2))
    weights, offsets = torch.full((T, k), math.nan, device="cuda"), torch.full((E + 1,), -1, dtype=torch.int32, device="cuda")
    route = cc.Route(T, E, k, 0, stream(), VT.float16)
    route.Run(logits.data_ptr(), experts.data_ptr(), weights.data_ptr(), offsets.data_ptr(), slots.data_ptr())
    want = torch.stack([(E - 1 - rows) * 73 % E, (E - 2 - rows) * 73 % E], dim=1)
    assert torch.equal(experts.long(), want)
    assert torch.equal(offsets[1:].long(), torch.bincount(want.flatten(), minlength=E).cumsum(0)) and int(offsets[0]) == 0
    order = torch.sort(want.flatten(), stable=True).indices
    assert torch.equal(slots.flatten()[order].long(), torch.arange(T * k, device="cuda"))
    p = 1 / (1 + math.exp(-1.0))
    error = (88 + 8 + E) * 2.0 ** -23                       # (as check_route's)
    assert float((weights.double() - torch.tensor([p, 1 - p], dtype=torch.float64, device="cuda")).abs().max()) <= error
    dweights = torch.tensor([3.0, -1.0], device="cuda").repeat(T, 1)
    dlogits = logits.fill_(math.nan)                        # (logits are not read where the weights are of the chosen alone)
    route.Backward(0, experts.data_ptr(), weights.data_ptr(), dweights.data_ptr(), dlogits.data_ptr())
    size = p * (1 - p) * 4.0                                # w_0 (dw_0 - (w_0 dw_0 + w_1 dw_1)), and the second is its opposite
    for at in range(0, T, step):
        full = torch.zeros((min(step, T - at), E), dtype=torch.float64, device="cuda")
        full.scatter_(1, want[at:at + step], torch.tensor([size, -size], dtype=torch.float64, device="cuda").repeat(len(full), 1))
        assert float((dlogits[at:at + step].double() - full).abs().max()) <= 8 * error + 2.0 ** -11 * size


def test_combine_beyond_32_bits():
    """Rows 8 MiB apart, 5 GB of each operand."""
    run_combine(600, 1, 40, VT.bfloat16, 610, True, 1 << 22, 1 << 22, holes=True)


@pytest.mark.parametrize("t", list(TORCH))
def test_the_smallest_differences(t):
    """Neighbouring values, among them the smallest above and below zero, and both infinities: bits decide."""
    info = torch.finfo(TORCH[t])
    step = {VT.float16: 2.0 ** -24, VT.bfloat16: 2.0 ** -133, VT.float32: 2.0 ** -149}[t]
    values = [0.0, -0.0, step, -step, 2 * step, -2 * step, info.tiny, -info.tiny, info.max, -info.max, math.inf, -math.inf, 1.0,
              1.0 + info.eps, 1.0 - info.eps / 2, -1.0]
    assert len(set(torch.tensor(values, dtype=TORCH[t]).tolist())) == len(values) - 1          # (the zeros)
    gen = torch.Generator().manual_seed(3)
    logits = torch.stack([torch.tensor(values, dtype=TORCH[t])[torch.randperm(len(values), generator=gen)] for _ in range(200)])
    for k in (3, 16):
        experts, _, offsets, slots, _, _ = run_route(logits, k, True)
        e, _, o, s = routed(logits, k, True)
        assert torch.equal(experts.long(), e) and offsets.tolist() == o and torch.equal(slots.long(), s)


@pytest.mark.parametrize("t", list(HALF))
def test_masks_and_values_that_are_not_finite_of_16_bits(t):
    gen = torch.Generator().manual_seed(1)
    logits = torch.randn((40, 300), generator=gen)
    logits[:, 5:280] = -math.inf
    logits[3] = -math.inf
    logits[6] = torch.finfo(HALF[t]).min
    for normalize in (True, False):
        check_route(logits.to(HALF[t]), 16, normalize)
        check_route(logits[:, :30].to(HALF[t]), 12, normalize)
    logits = torch.zeros((4, 20))
    logits[0, 7], logits[0, 3], logits[1], logits[2, 11] = math.nan, math.inf, math.nan, math.inf
    experts, weights, _, _, _, _ = run_route(logits.to(HALF[t]), 3, True)
    assert experts.tolist() == [[7, 3, 0], [0, 1, 2], [11, 0, 1], [0, 1, 2]]
    assert bool(weights[:3].isnan().any(dim=1).all()) and not bool(weights[3].isnan().any())
