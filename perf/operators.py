"""The work that the 8-bit products with block scales and the orthogonalised updates are measured on.

A case is a dict of plain values. `path` says which operator it goes through:

    quantize       Quantize: B matrices of M x N to 8 bits with a scale for each group of 128 ("rows": 128 values of a
                   row, "blocks": 128 x 128 values), as they are, or also their transposes ("both")
    product        ScaledGEMM: C [M][N] (+)= A [M][K] B [N][K]^T of such operands
    linear         ScaledLinear: weights laid out, forward and backward of a layer of K inputs and N outputs on M rows
    orthogonalize  Orthogonalize: Newton-Schulz steps on B updates of M x N

The plain form of each is made of elementary torch operations in 32 bits, rounded once at the end.
"""
import math

import torch

own = False

F8 = {"float8e4m3": (torch.float8_e4m3fn, 448.0), "float8e5m2": (torch.float8_e5m2, 57344.0)}
TORCH = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
BYTES = {"float16": 2, "bfloat16": 2, "float32": 4}
GROUP = 128
SMALLEST = 2.0 ** -100                     # no group's largest value counts as less
STEPS, COEFFICIENTS, EPSILON = 5, (3.4445, -4.7750, 2.0315), 1e-7


def _up(n, to=16):
    return (n + to - 1) // to * to


def _quantize_case(B, M, N, tin, tout="float8e4m3", group="rows", scale="float32", both=False, name=None):
    case = {"path": "quantize", "B": B, "M": M, "N": N, "tin": tin, "tout": tout, "group": group, "scale": scale,
            "both": both}
    return dict(case, name=name) if name else case


def _product_case(B, M, N, K, ta="float8e4m3", tb="float8e4m3", tout="bfloat16", group_a="rows", group_b="blocks",
                  scale="float32", accumulate=False, name=None):
    case = {"path": "product", "B": B, "M": M, "N": N, "K": K, "ta": ta, "tb": tb, "tout": tout, "group_a": group_a,
            "group_b": group_b, "scale": scale, "accumulate": accumulate}
    return dict(case, name=name) if name else case


def _linear_case(M, N, K, t="bfloat16", tgrad="float8e5m2", scale="e8m0", name=None):
    case = {"path": "linear", "M": M, "N": N, "K": K, "t": t, "tgrad": tgrad, "scale": scale}
    return dict(case, name=name) if name else case


def _orthogonalize_case(B, M, N, t, name=None):
    case = {"path": "orthogonalize", "B": B, "M": M, "N": N, "t": t}
    return dict(case, name=name) if name else case


def listed():
    return [
        # One token's activations in front of a product: launch latency.
        _quantize_case(1, 1, 4096, "bfloat16", name="quantize_token"),
        # Activations of a training step, for the forward product and, transposed, for the weights' gradient; odd sizes.
        _quantize_case(1, 8191, 8200, "bfloat16", both=True, name="quantize_both_ways"),
        # One token against a layer's weights: the weights' bytes.
        _product_case(1, 1, 8192, 8192, name="product_token"),
        # A handful of small layers at once, sizes that fit no tile, scales that are powers of two.
        _product_case(16, 300, 577, 1000, tout="float32", scale="e8m0", name="product_ragged"),
        # A prompt or a training batch through a large layer.
        _product_case(1, 8192, 8192, 8192, name="product_8192"),
        # Gradient of weights, summed over an odd number of rows into 32 bits: scales along both operands' rows.
        _product_case(1, 4096, 2048, 8191, ta="float8e5m2", tout="float32", group_b="rows", accumulate=True,
                      name="product_weight_gradient"),
        # A small layer, forward and backward, from 32-bit values.
        _linear_case(300, 255, 576, t="float32", tgrad="float8e4m3", scale="float32", name="linear_small"),
        # A large one as it is trained.
        _linear_case(8192, 4096, 4096, name="linear_8192"),
        # The updates of many small matrices (heads, adapters) in one call.
        _orthogonalize_case(16, 128, 96, "bfloat16", name="orthogonalize_16_small"),
        # Two updates kept in 32 bits, sizes that fit no tile.
        _orthogonalize_case(2, 1000, 1000, "float32", name="orthogonalize_1000"),
        # A layer that narrows: more rows than columns.
        _orthogonalize_case(1, 4096, 1024, "bfloat16", name="orthogonalize_tall"),
        # The largest layer.
        _orthogonalize_case(1, 4096, 8192, "bfloat16", name="orthogonalize_large"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _extent(rng, low, high):
    """A size between low and high: as it falls, or rounded to a multiple that arrays often have."""
    step = rng.choice([1, 1, 8, 64, 128])
    n = 3072
    while n == 3072:                       # (a size that nothing here has)
        n = _log(rng, low, high)
        n = max(low, min(high, (n + step // 2) // step * step))
    return n


def draw(rng):
    """One case of the ranges the listed ones stand for."""
    path = rng.choice(["quantize", "product", "product", "linear", "orthogonalize", "orthogonalize"])
    scale = rng.choice(["float32", "float32", "e8m0"])
    while True:
        if path == "quantize":
            case = _quantize_case(_log(rng, 1, 16), _extent(rng, 1, 8192), _extent(rng, 16, 8192),
                                  rng.choice(["bfloat16", "bfloat16", "float16", "float32"]),
                                  rng.choice(["float8e4m3", "float8e4m3", "float8e5m2"]),
                                  rng.choice(["rows", "rows", "blocks"]), scale, rng.random() < 0.5)
        elif path == "product":
            case = _product_case(_log(rng, 1, 16), _extent(rng, 1, 8192), _extent(rng, 16, 8192), _extent(rng, 16, 8192),
                                 rng.choice(["float8e4m3", "float8e4m3", "float8e5m2"]), "float8e4m3",
                                 rng.choice(["bfloat16", "bfloat16", "float16", "float32"]),
                                 "rows", rng.choice(["rows", "blocks", "blocks"]), scale, rng.random() < 0.2)
            if case["accumulate"]:
                case["tout"] = "float32"
        elif path == "linear":
            case = _linear_case(_extent(rng, 16, 8192), _extent(rng, 16, 8192), _extent(rng, 16, 8192),
                                rng.choice(["bfloat16", "bfloat16", "float16", "float32"]),
                                rng.choice(["float8e4m3", "float8e5m2"]), scale)
        else:
            case = _orthogonalize_case(_log(rng, 1, 16), _extent(rng, 16, 8192), _extent(rng, 16, 8192),
                                       rng.choice(["bfloat16", "bfloat16", "float16", "float32"]))
        w = work(case)
        if w["bytes"] <= 1e9 and w["flops"] <= (1.0e12 if path != "orthogonalize" else 6e11):
            return case


def _activations(shape, gen, outliers=1.0):
    """N(0, 1) values whose columns differ in size, a few of them by a lot."""
    x = torch.randn(shape, device="cuda", generator=gen)
    spread = torch.exp(torch.randn(shape[-1], device="cuda", generator=gen) * 0.5)
    spread[:: 97] *= 1.0 + 20.0 * outliers
    return x * spread


def _gradients(shape, gen):
    """Small values whose rows (tokens) differ in size by orders of magnitude."""
    x = torch.randn(shape, device="cuda", generator=gen)
    return x * torch.exp(torch.randn(shape[:-1] + (1,), device="cuda", generator=gen) * 1.5) * 1e-3


def _update(B, M, N, gen):
    """Momentum of a weight matrix: some directions that persist over noise."""
    k = max(1, min(M, N) // 8)
    low = torch.randn((B, M, k), device="cuda", generator=gen) @ torch.randn((B, k, N), device="cuda", generator=gen)
    return (low / math.sqrt(k) + torch.randn((B, M, N), device="cuda", generator=gen)) * 1e-3


# ---- plain forms ---------------------------------------------------------------------------------------------------

def _largest(x, group):
    """Largest finite magnitude of each group of x [B][R][C]: [B][R or R/128][C/128]."""
    B, R, C = x.shape
    x = x.abs()
    x = torch.where(torch.isfinite(x), x, torch.zeros_like(x))
    g = _up(C, GROUP) // GROUP
    x = torch.nn.functional.pad(x, (0, g * GROUP - C)).view(B, R, g, GROUP).amax(dim=3)
    if group == "blocks":
        r = _up(R, GROUP) // GROUP
        x = torch.nn.functional.pad(x, (0, 0, 0, r * GROUP - R)).view(B, r, GROUP, g).amax(dim=2)
    return x.clamp(min=SMALLEST)


def _spread(s, group, R, C):
    """A factor for each value from one for each group [B][rows][C/128]."""
    s = s.repeat_interleave(GROUP, dim=2)[:, :, :C]
    return s.repeat_interleave(GROUP, dim=1)[:, :R] if group == "blocks" else s


def _power_of_two_from(r):
    """Exponent of the smallest power of two that is no less than r (32 bits)."""
    m, e = torch.frexp(r)
    return torch.where(m == 0.5, e - 1, e)


def _power_of_two(e):
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _plain_quantize(x, tout, group, scale):
    """Values of 8 bits [B][R][C] and scales [B][C/128][rows or rows/128] (32 bits) of x [B][R][C] (32 bits)."""
    dtype, top = F8[tout]
    amax = _largest(x, group)
    top = torch.full_like(amax, top)       # (a tensor: torch divides by a number by multiplying with its reciprocal)
    if scale == "e8m0":
        e = _power_of_two_from(amax / top)
        s, inverse = _power_of_two(e), _power_of_two(-e)
    else:
        s, inverse = amax / top, top / amax
    q = (x * _spread(inverse, group, x.shape[1], x.shape[2])).to(dtype)
    return q, s.transpose(1, 2).contiguous()


def _as_scales(s, scale):
    return s.to(torch.float8_e8m0fnu) if scale == "e8m0" else s


def _plain_values(q, s, group):
    """What 8-bit values [B][R][C] with scales [B][C/128][rows] stand for, in 32 bits."""
    return q.float() * _spread(s.float().transpose(1, 2), group, q.shape[1], q.shape[2])


def _through_8_bits(x, tout, group, scale):
    q, s = _plain_quantize(x, tout, group, scale)
    return _plain_values(q, s, group)


def _plain_orthogonalize(g):
    a, b, c = COEFFICIENTS
    tall = g.shape[1] > g.shape[2]
    x = (g.transpose(1, 2) if tall else g).contiguous().float()
    x = x / (torch.sqrt((x * x).sum(dim=(1, 2), keepdim=True)) + EPSILON)
    for _ in range(STEPS):
        s = torch.bmm(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.bmm(b * s + c * torch.bmm(s, s), x)
    return (x.transpose(1, 2) if tall else x).to(g.dtype)


def _plain(state):
    case = state["case"]
    path = case["path"]
    if path == "quantize":
        x = state["x"].float()
        q, s = _plain_quantize(x, case["tout"], case["group"], case["scale"])
        out = {"q": q, "scales": _as_scales(s, case["scale"])}
        if case["both"]:
            q, s = _plain_quantize(x.transpose(1, 2).contiguous(), case["tout"], case["group"], case["scale"])
            out |= {"q_t": q, "scales_t": _as_scales(s, case["scale"])}
        return out
    if path == "product":
        a = _plain_values(state["a"][:, :, :case["K"]], state["sa"][:, :, :state["rows_a"]], case["group_a"])
        b = _plain_values(state["b"][:, :, :case["K"]], state["sb"][:, :, :state["rows_b"]], case["group_b"])
        c = torch.bmm(a, b.transpose(1, 2).contiguous())
        if case["accumulate"]:
            return {"c": state["c"].add_(c)}
        return {"c": c.to(state["c"].dtype)}
    if path == "linear":
        x, w, dy = (state[k].float()[None] for k in ("x", "w", "dy"))
        scale, tg, t = case["scale"], case["tgrad"], state["x"].dtype
        y = _through_8_bits(x, "float8e4m3", "rows", scale)[0] @ _through_8_bits(w, "float8e4m3", "blocks", scale)[0].t()
        dx = (_through_8_bits(dy, tg, "rows", scale)[0]
              @ _through_8_bits(w.transpose(1, 2).contiguous(), "float8e4m3", "blocks", scale)[0].t())
        dw = (_through_8_bits(dy.transpose(1, 2).contiguous(), tg, "rows", scale)[0]
              @ _through_8_bits(x.transpose(1, 2).contiguous(), "float8e4m3", "rows", scale)[0].t())
        return {"y": y.to(t), "dx": dx.to(t), "dw": dw}
    return {"out": _plain_orthogonalize(state["g"])}


# ---- the framework's operators -------------------------------------------------------------------------------------

_plans = {}                                # one object for each size, as a program with such layers keeps


def _plan(state):
    import ccglib_amd as cc
    case, stream = state["case"], torch.cuda.current_stream().cuda_stream
    key = (stream,) + tuple(v for k, v in case.items() if k != "name")
    plan = _plans.get(key)
    if plan is not None:
        return plan
    vt, st, sg, path = cc.ValueType, cc.ScaleType, cc.ScaleGroup, case["path"]
    if path == "quantize":
        plan = cc.Quantize(case["B"], case["M"], case["N"], 0, stream, vt[case["tin"]], vt[case["tout"]],
                           sg[case["group"]], st[case["scale"]])
    elif path == "product":
        plan = cc.ScaledGEMM(case["B"], case["M"], case["N"], case["K"], 0, stream, vt[case["ta"]], vt[case["tb"]],
                             vt[case["tout"]], sg[case["group_a"]], sg[case["group_b"]], st[case["scale"]],
                             case["accumulate"])
    elif path == "linear":
        plan = cc.ScaledLinear(case["M"], case["N"], case["K"], 0, stream, vt[case["t"]], vt[case["tgrad"]],
                               st[case["scale"]])
    else:
        plan = cc.Orthogonalize(case["B"], case["M"], case["N"], 0, stream, vt[case["t"]], STEPS, COEFFICIENTS, EPSILON)
    _plans[key] = plan
    return plan


def _own(state):
    case, plan = state["case"], _plan(state)
    path = case["path"]
    if path == "quantize":
        both = case["both"]
        plan.Run(state["x"].data_ptr(), state["q"].data_ptr(), state["s"].data_ptr(),
                 state["qt"].data_ptr() if both else 0, state["st"].data_ptr() if both else 0)
        M, N = case["M"], case["N"]
        rows, cols = (M, N) if case["group"] == "rows" else (_up(M, GROUP) // GROUP, _up(N, GROUP) // GROUP)
        out = {"q": state["q"][:, :, :N], "scales": state["s"][:, :, :rows]}
        if both:
            out |= {"q_t": state["qt"][:, :, :M], "scales_t": state["st"][:, :, :cols]}
        return out
    if path == "product":
        plan.Run(state["a"].data_ptr(), state["sa"].data_ptr(), state["b"].data_ptr(), state["sb"].data_ptr(),
                 state["c"].data_ptr())
        return {"c": state["c"]}
    if path == "linear":
        plan.SetWeights(state["w"].data_ptr())
        plan.Forward(state["x"].data_ptr(), state["y"].data_ptr())
        plan.Backward(state["dy"].data_ptr(), state["dx"].data_ptr(), state["dw"].data_ptr())
        return {"y": state["y"], "dx": state["dx"], "dw": state["dw"]}
    plan.Run(state["g"].data_ptr(), state["out"].data_ptr())
    return {"out": state["out"]}


def _operand(B, rows, K, t, group, scale, gen, gradient):
    """An operand of a product as a program holds it: rows of 8-bit values padded to 16 bytes with zeros, scales with
    the groups of K outermost, their rows padded to 16."""
    x = _gradients((B, rows, K), gen) if gradient else _activations((B, rows, K), gen)
    q, s = _plain_quantize(x, t, group, scale)
    held = torch.zeros((B, rows, _up(K)), dtype=torch.uint8, device="cuda")
    held[:, :, :K] = q.view(torch.uint8)
    s = torch.nn.functional.pad(s, (0, _up(s.shape[2]) - s.shape[2]), value=1.0)
    return held.view(F8[t][0]), _as_scales(s, scale)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    path, M, N = case["path"], case["M"], case["N"]
    state = {"case": dict(case)}
    if path == "quantize":
        B, dtype = case["B"], F8[case["tout"]][0]
        state["x"] = _activations((B, M, N), gen).to(TORCH[case["tin"]])
        sdtype = torch.float8_e8m0fnu if case["scale"] == "e8m0" else torch.float32
        for q, s, rows, cols in (("q", "s", M, N), ("qt", "st", N, M)):
            if q == "qt" and not case["both"]:
                continue
            groups = rows if case["group"] == "rows" else _up(rows, GROUP) // GROUP
            state[q] = torch.empty((B, rows, _up(cols)), dtype=dtype, device="cuda")
            state[s] = torch.empty((B, _up(cols, GROUP) // GROUP, _up(groups)), dtype=sdtype, device="cuda")
    elif path == "product":
        B, K = case["B"], case["K"]
        state["a"], state["sa"] = _operand(B, M, K, case["ta"], case["group_a"], case["scale"], gen, case["accumulate"])
        state["b"], state["sb"] = _operand(B, N, K, case["tb"], case["group_b"], case["scale"], gen, False)
        for rows, n, g in (("rows_a", M, case["group_a"]), ("rows_b", N, case["group_b"])):
            state[rows] = n if g == "rows" else _up(n, GROUP) // GROUP
        c = torch.randn((B, M, N), device="cuda", generator=gen) if case["accumulate"] else torch.empty(
            (B, M, N), device="cuda")
        state["c"] = c.to(TORCH[case["tout"]])
    elif path == "linear":
        K, t = case["K"], TORCH[case["t"]]
        state["x"] = _activations((M, K), gen).to(t)
        state["w"] = (torch.randn((N, K), device="cuda", generator=gen) / math.sqrt(K)).to(t)
        state["dy"] = _gradients((M, N), gen).to(t)
        state["y"], state["dx"] = torch.empty((M, N), dtype=t, device="cuda"), torch.empty((M, K), dtype=t, device="cuda")
        state["dw"] = torch.empty((N, K), dtype=torch.float32, device="cuda")
    else:
        state["g"] = _update(case["B"], M, N, gen).to(TORCH[case["t"]])
        state["out"] = torch.empty_like(state["g"])
    return state


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    path, M, N = case["path"], case["M"], case["N"]
    width = {"float32": 4, "e8m0": 1}

    def scales(rows, cols, group, scale):
        return _up(cols, GROUP) // GROUP * (rows if group == "rows" else _up(rows, GROUP) // GROUP) * width[scale]

    if path == "quantize":
        size = M * N * BYTES[case["tin"]] + M * N + scales(M, N, case["group"], case["scale"])
        if case["both"]:
            size += M * N + scales(N, M, case["group"], case["scale"])
        return {"bytes": case["B"] * size, "flops": 0}
    if path == "product":
        K = case["K"]
        size = ((M + N) * K + scales(M, K, case["group_a"], case["scale"]) + scales(N, K, case["group_b"], case["scale"])
                + M * N * BYTES[case["tout"]] * (2 if case["accumulate"] else 1))
        return {"bytes": case["B"] * size, "flops": 2 * case["B"] * M * N * K}
    if path == "linear":
        K, size = case["K"], BYTES[case["t"]]
        # x, w and dy come in, y and dx go out, dw goes out in 32 bits
        return {"bytes": size * (2 * M * K + N * K + 2 * M * N) + 4 * N * K, "flops": 6 * M * N * K}
    m, n = min(M, N), max(M, N)
    # (X X^T and its square are symmetric: half of each)
    return {"bytes": case["B"] * 2 * M * N * BYTES[case["t"]],
            "flops": case["B"] * STEPS * (m * m * n + m * m * m + 2 * m * m * n)}


# ---- 64 bits -------------------------------------------------------------------------------------------------------

def _expand(s, rows, cols, group_rows):
    """s [B][K/128][groups] in 64 bits -> [B][rows][cols], by indexing."""
    r = torch.arange(rows, device="cuda") // group_rows
    k = torch.arange(cols, device="cuda") // GROUP
    return s.double()[:, k][:, :, r].transpose(1, 2)


def _quantize_64(x, tout, group, scale):
    """(8-bit values and scales, both in 64 bits, [B][R][C] and [B][C/128][groups]) from the definition: the factor and
    the scale are numbers of 32 bits, the product with the factor is rounded once, to 8 bits."""
    dtype, top = F8[tout]
    B, R, C = x.shape
    x = x.double()
    rows = 1 if group == "rows" else GROUP
    R_groups, C_groups = -(-R // rows), -(-C // GROUP)
    padded = torch.zeros((B, R_groups * rows, C_groups * GROUP), dtype=torch.float64, device="cuda")
    padded[:, :R, :C] = x.abs()
    amax = padded.reshape(B, R_groups, rows, C_groups, GROUP).amax(dim=(2, 4)).clamp(min=SMALLEST).transpose(1, 2)
    if scale == "e8m0":
        s = torch.exp2(torch.ceil(torch.log2((amax / top).float().double())))
        inverse = 1.0 / s
    else:
        s, inverse = (amax / top).float().double(), (top / amax).float().double()
    q = (x * _expand(inverse, R, C, rows)).float().to(dtype).double()
    return q, s


def _values_64(x, tout, group, scale):
    q, s = _quantize_64(x, tout, group, scale)
    return q * _expand(s, q.shape[1], q.shape[2], 1 if group == "rows" else GROUP)


def exact(case, seed):
    """What run() returns for these inputs, in 64 bits."""
    state = prepare(case, seed)
    path = case["path"]
    if path == "quantize":
        q, s = _quantize_64(state["x"], case["tout"], case["group"], case["scale"])
        out = {"q": q, "scales": s}
        if case["both"]:
            q, s = _quantize_64(state["x"].transpose(1, 2), case["tout"], case["group"], case["scale"])
            out |= {"q_t": q, "scales_t": s}
        return out
    if path == "product":
        M, N, K = case["M"], case["N"], case["K"]
        c = state["c"].double() if case["accumulate"] else torch.zeros(state["c"].shape, dtype=torch.float64, device="cuda")
        rows_a, rows_b = (1 if case[g] == "rows" else GROUP for g in ("group_a", "group_b"))
        for i in range(case["B"]):
            a = state["a"][i:i + 1, :, :K].float().double() * _expand(state["sa"][i:i + 1].float(), M, K, rows_a)
            b = state["b"][i:i + 1, :, :K].float().double() * _expand(state["sb"][i:i + 1].float(), N, K, rows_b)
            c[i] += a[0] @ b[0].t().contiguous()
        return {"c": c}
    if path == "linear":
        x, w, dy = (state[k][None] for k in ("x", "w", "dy"))
        scale, tg, e4m3 = case["scale"], case["tgrad"], "float8e4m3"
        y = _values_64(x, e4m3, "rows", scale)[0] @ _values_64(w, e4m3, "blocks", scale)[0].t().contiguous()
        dx = _values_64(dy, tg, "rows", scale)[0] @ _values_64(w, e4m3, "blocks", scale)[0]
        dw = (_values_64(dy.transpose(1, 2), tg, "rows", scale)[0]
              @ _values_64(x.transpose(1, 2), e4m3, "rows", scale)[0].t().contiguous())
        return {"y": y, "dx": dx, "dw": dw}
    a, b, c = COEFFICIENTS
    out = []
    for g in state["g"].double():
        x = g / (torch.linalg.matrix_norm(g) + EPSILON)
        for _ in range(STEPS):       # (on the side of the shorter extent: both give the same polynomial of x)
            if x.shape[0] <= x.shape[1]:
                s = x @ x.t().contiguous()
                x = a * x + (b * s + c * (s @ s)) @ x
            else:
                s = x.t().contiguous() @ x
                x = a * x + x @ (b * s + c * (s @ s))
        out.append(x)
    return {"out": torch.stack(out)}
