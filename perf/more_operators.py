"""The work that the 16-bit linear layers, those grouped by expert, and the routing between them are measured on.

A case is a dict of plain values. `path` says which operator it goes through:

    linear            FusedLinear, forward: z = x W^T + b, y = act(z) + r
    linear_gradient   FusedLinear, backward: dz = dy act'(z), dx = dz W, dW (+)= dz^T x, db (+)= column sums of dz
    grouped           GroupedLinear, forward: the same with a W and a b for each expert, rows sorted by expert
    grouped_gradient  GroupedLinear, backward
    route             Route: the k largest of E logits a token, their weights, and where each token's rows lie when all
                      rows are sorted by expert; with the logits' gradient
    combine           Combine: sums of the k rows of a token with their weights, or (gradient) their gradients

The plain form of each is made of elementary torch operations in 32 bits, rounded once at the end.
"""
import math

import torch

own = False

TORCH = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
BYTES = {"float16": 2, "bfloat16": 2, "float32": 4}
GELU = math.sqrt(2.0 / math.pi), 0.044715


def _linear_case(M, N, K, t="bfloat16", activation="none", bias=True, residual=False, keep=False, name=None):
    case = {"path": "linear", "M": M, "N": N, "K": K, "t": t, "activation": activation, "bias": bias,
            "residual": residual, "keep": keep}
    return dict(case, name=name) if name else case


def _linear_gradient_case(M, N, K, t="bfloat16", activation="none", tgrad="bfloat16", accumulate=False, name=None):
    case = {"path": "linear_gradient", "M": M, "N": N, "K": K, "t": t, "activation": activation, "tgrad": tgrad,
            "accumulate": accumulate}
    return dict(case, name=name) if name else case


def _grouped_case(E, M, N, K, t="bfloat16", activation="none", bias=False, name=None):
    case = {"path": "grouped", "E": E, "M": M, "N": N, "K": K, "t": t, "activation": activation, "bias": bias}
    return dict(case, name=name) if name else case


def _grouped_gradient_case(E, M, N, K, t="bfloat16", activation="none", tgrad="bfloat16", name=None):
    case = {"path": "grouped_gradient", "E": E, "M": M, "N": N, "K": K, "t": t, "activation": activation,
            "tgrad": tgrad, "accumulate": False}
    return dict(case, name=name) if name else case


def _route_case(T, E, k, t="float32", normalize=True, name=None):
    case = {"path": "route", "T": T, "E": E, "k": k, "t": t, "normalize": normalize}
    return dict(case, name=name) if name else case


def _combine_case(T, k, N, t="bfloat16", gradient=False, name=None):
    case = {"path": "combine", "T": T, "k": k, "N": N, "t": t, "gradient": gradient}
    return dict(case, name=name) if name else case


def listed():
    return [
        # One token through a layer: the weights' bytes.
        _linear_case(1, 8192, 8192, activation="silu", name="linear_token"),
        # A short prompt through a small layer of sizes that fit no tile.
        _linear_case(300, 577, 1000, t="float16", activation="gelu", residual=True, name="linear_ragged"),
        # A prompt or a training batch through a large layer, its pre-activations kept for the backward pass.
        _linear_case(8192, 8192, 8192, activation="gelu", residual=True, keep=True, name="linear_8192"),
        # Gradients of a small layer of odd sizes, the weights' and the bias' summed into 32 bits.
        _linear_gradient_case(300, 255, 577, t="float16", tgrad="float32", accumulate=True, name="linear_gradient_ragged"),
        # A large one as it is trained.
        _linear_gradient_case(8192, 4096, 4096, activation="silu", name="linear_gradient_8192"),
        # Eight tokens, two experts each, out of 64: the weights' bytes of those that are asked.
        _grouped_case(64, 16, 2048, 2048, activation="silu", name="grouped_tokens"),
        # A prompt through sixteen experts, some of them with few rows, one with none.
        _grouped_case(16, 16383, 4096, 2048, activation="silu", bias=True, name="grouped_prompt"),
        # Experts as they are trained.
        _grouped_gradient_case(16, 8192, 4096, 2048, activation="gelu", name="grouped_gradient_8192"),
        # A handful of tokens: launch latency.
        _route_case(8, 64, 2, t="bfloat16", name="route_tokens"),
        # A training batch.
        _route_case(65536, 128, 8, normalize=False, name="route_65536"),
        # A prompt's rows back to its tokens; odd sizes.
        _combine_case(4099, 2, 4104, t="float16", name="combine_ragged"),
        # Gradients of a training batch's rows and weights.
        _combine_case(16384, 4, 4096, gradient=True, name="combine_gradient_16384"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _extent(rng, low, high):
    """A size between low and high: as it falls, or rounded to a multiple that arrays often have."""
    step = rng.choice([1, 1, 8, 64, 128])
    n = _log(rng, low, high)
    return max(low, min(high, (n + step // 2) // step * step))


def draw(rng):
    """One case of the ranges the listed ones stand for."""
    path = rng.choice(["linear", "linear", "linear_gradient", "grouped", "grouped_gradient", "route", "combine"])
    t = rng.choice(["bfloat16", "bfloat16", "float16"])
    activation = rng.choice(["none", "relu", "gelu", "silu"])
    while True:
        M, N, K, E = _extent(rng, 1, 8192), _extent(rng, 16, 8192), _extent(rng, 16, 8192), _log(rng, 2, 128)
        if path == "linear":
            case = _linear_case(M, N, K, t, activation, rng.random() < 0.7, rng.random() < 0.4, rng.random() < 0.3)
        elif path == "linear_gradient":
            case = _linear_gradient_case(max(M, 16), N, K, t, activation, t)
            if activation == "none" and rng.random() < 0.5:
                case = dict(case, tgrad="float32", accumulate=True)
        elif path == "grouped":
            case = _grouped_case(E, 2 * M, N, K, t, activation, rng.random() < 0.5)
        elif path == "grouped_gradient":
            case = _grouped_gradient_case(E, 2 * max(M, 16), N, K, t, activation, t)
        elif path == "route":
            E = _extent(rng, 4, 512)
            case = _route_case(_extent(rng, 1, 65536), E, min(E, _log(rng, 1, 8)), rng.choice(["float32", t]),
                               rng.random() < 0.5)
        else:
            case = _combine_case(_extent(rng, 1, 32768), _log(rng, 1, 8), N, t, rng.random() < 0.5)
        w = work(case)
        if w["bytes"] <= 1e9 and w["flops"] <= 5e11:
            return case


def _activations(shape, gen):
    """N(0, 1) values whose columns differ in size."""
    return (torch.randn(shape, device="cuda", generator=gen)
            * torch.exp(torch.randn(shape[-1], device="cuda", generator=gen) * 0.5))


def _gradients(shape, gen):
    """Small values whose rows (tokens) differ in size."""
    return (torch.randn(shape, device="cuda", generator=gen)
            * torch.exp(torch.randn(shape[:-1] + (1,), device="cuda", generator=gen)) * 1e-2)


# ---- plain forms ---------------------------------------------------------------------------------------------------

def _sigmoid(a):
    return 1.0 / (1.0 + torch.exp(-a))


def _gelu_gate(z):
    """The gate g of gelu(z) = z g, 1/2 (1 + tanh(a)) with a = sqrt(2/pi) (z + 0.044715 z^3), and d(2 a)/dz."""
    c, d = GELU
    return _sigmoid(2.0 * c * (z + d * z * z * z)), 2.0 * c * (1.0 + 3.0 * d * z * z)


def _act(z, activation):
    if activation == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if activation == "gelu":
        return z * _gelu_gate(z)[0]
    return z * _sigmoid(z) if activation == "silu" else z


def _act_gradient(z, activation):
    if activation == "relu":
        return (z > 0).to(z.dtype)
    if activation == "gelu":
        g, slope = _gelu_gate(z)
        return g + z * g * (1.0 - g) * slope
    if activation == "silu":
        g = _sigmoid(z)
        return g + z * g * (1.0 - g)
    return torch.ones_like(z)


def _plain_linear(state, case, x, w, b, r):
    """z and y of a layer, 32 bits."""
    z = x.float() @ w.float().t()
    if b is not None:
        z = z + b.float()
    y = _act(z, case["activation"])
    return z, (y if r is None else y + r.float())


def _plain_gradients(case, dy, z, x, w):
    """dx, dw, db of a layer, 32 bits."""
    dz = dy.float() * _act_gradient(z.float(), case["activation"])
    return dz @ w.float(), dz.t().contiguous() @ x.float(), dz.sum(dim=0)


def _plain_route(state, case):
    logits, k, E = state["logits"], case["k"], case["E"]
    chosen, experts = torch.sort(logits, dim=1, descending=True, stable=True)
    chosen, experts = chosen[:, :k].float(), experts[:, :k].contiguous()
    every = logits.float()
    top = every.amax(dim=1, keepdim=True)
    scale = torch.exp(chosen - top).sum(dim=1, keepdim=True) if case["normalize"] else torch.exp(every - top).sum(dim=1, keepdim=True)
    weights = torch.exp(chosen - top) / scale
    order = torch.argsort(experts.flatten(), stable=True)
    slots = torch.empty_like(order)
    slots[order] = torch.arange(order.numel(), device=order.device)
    counts = (experts.flatten()[None, :] == torch.arange(E, device=order.device)[:, None]).sum(dim=1)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    inner = (weights * state["dweights"]).sum(dim=1, keepdim=True)
    if case["normalize"]:
        dlogits = torch.zeros_like(every).scatter_(1, experts, weights * (state["dweights"] - inner))
    else:
        p = torch.exp(every - top) / scale
        dlogits = (p * -inner).scatter_add_(1, experts, weights * state["dweights"])
    return {"experts": experts.to(torch.int32), "weights": weights, "offsets": offsets.to(torch.int32),
            "slots": slots.view_as(experts).to(torch.int32), "dlogits": dlogits.to(logits.dtype)}


def _plain(state):
    case = state["case"]
    path = case["path"]
    if path == "linear":
        t = state["x"].dtype
        z, y = _plain_linear(state, case, state["x"], state["w"], state["b"], state["r"])
        return {"y": y.to(t), "z": z.to(t)} if case["keep"] else {"y": y.to(t)}
    if path == "linear_gradient":
        dx, dw, db = _plain_gradients(case, state["dy"], state["z"], state["x"], state["w"])
        if case["accumulate"]:
            return {"dx": dx.to(state["x"].dtype), "dw": state["dw"].add_(dw), "db": state["db"].add_(db)}
        return {"dx": dx.to(state["x"].dtype), "dw": dw.to(state["dw"].dtype), "db": db.to(state["db"].dtype)}
    if path == "grouped":
        o, y = state["starts"], state["y"]
        for e in range(case["E"]):
            b = None if state["b"] is None else state["b"][e]
            y[o[e]:o[e + 1]] = _plain_linear(state, case, state["x"][o[e]:o[e + 1]], state["w"][e], b, None)[1].to(y.dtype)
        return {"y": y}
    if path == "grouped_gradient":
        o, out = state["starts"], {k: state[k] for k in ("dx", "dw", "db")}
        for e in range(case["E"]):
            rows = slice(o[e], o[e + 1])
            dx, dw, db = _plain_gradients(case, state["dy"][rows], state["z"][rows], state["x"][rows], state["w"][e])
            out["dx"][rows], out["dw"][e], out["db"][e] = dx.to(out["dx"].dtype), dw.to(out["dw"].dtype), db.to(out["db"].dtype)
        return out
    if path == "route":
        return _plain_route(state, case)
    y, slots, weights = state["y"], state["slots"].long(), state["weights"]
    rows = y[slots].float()                                              # [T][k][N]
    if case["gradient"]:
        d = state["dout"].float()
        dy = torch.empty_like(y)
        dy[slots] = (d[:, None, :] * weights[:, :, None]).to(y.dtype)
        return {"dy": dy, "dweights": (rows * d[:, None, :]).sum(dim=2)}
    return {"out": (rows * weights[:, :, None]).sum(dim=1).to(y.dtype)}


# ---- the framework's operators -------------------------------------------------------------------------------------

_plans = {}                                # one object for each size, as a program with such layers keeps


def _plan(state):
    import ccglib_amd as cc
    case, stream = state["case"], torch.cuda.current_stream().cuda_stream
    key = (stream,) + tuple(v for k, v in case.items() if k != "name")
    plan = _plans.get(key)
    if plan is not None:
        return plan
    vt, path = cc.ValueType, case["path"]
    if path.startswith("linear"):
        plan = cc.FusedLinear(case["M"], case["N"], case["K"], 0, stream, vt[case["t"]],
                              cc.Activation[case["activation"]], vt[case.get("tgrad", case["t"])],
                              training=path == "linear_gradient")
    elif path.startswith("grouped"):
        plan = cc.GroupedLinear(case["E"], case["M"], case["N"], case["K"], 0, stream, vt[case["t"]],
                                cc.Activation[case["activation"]], vt[case.get("tgrad", case["t"])],
                                training=path == "grouped_gradient")
    elif path == "route":
        plan = cc.Route(case["T"], case["E"], case["k"], 0, stream, vt[case["t"]], case["normalize"])
    else:
        plan = cc.Combine(case["T"], case["k"], case["N"], 0, stream, vt[case["t"]])
    _plans[key] = plan
    return plan


def _at(t):
    return 0 if t is None else t.data_ptr()


def _own(state):
    case, plan = state["case"], _plan(state)
    path = case["path"]
    if path == "linear":
        plan.Forward(_at(state["x"]), _at(state["w"]), _at(state["b"]), _at(state["r"]), _at(state["y"]), _at(state["z"]))
        return {"y": state["y"], "z": state["z"]} if case["keep"] else {"y": state["y"]}
    if path == "linear_gradient":
        plan.Backward(_at(state["dy"]), _at(state["z"]), _at(state["x"]), _at(state["w"]), _at(state["dx"]),
                      _at(state["dw"]), _at(state["db"]), accumulate=case["accumulate"])
        return {"dx": state["dx"], "dw": state["dw"], "db": state["db"]}
    if path == "grouped":
        plan.Forward(_at(state["x"]), _at(state["offsets"]), _at(state["w"]), _at(state["b"]), 0, _at(state["y"]), 0)
        return {"y": state["y"]}
    if path == "grouped_gradient":
        plan.Backward(_at(state["dy"]), _at(state["z"]), _at(state["x"]), _at(state["offsets"]), _at(state["w"]),
                      _at(state["dx"]), _at(state["dw"]), _at(state["db"]))
        return {"dx": state["dx"], "dw": state["dw"], "db": state["db"]}
    if path == "route":
        plan.Run(_at(state["logits"]), _at(state["experts"]), _at(state["weights"]), _at(state["offsets"]), _at(state["slots"]))
        plan.Backward(_at(state["logits"]), _at(state["experts"]), _at(state["weights"]), _at(state["dweights"]), _at(state["dlogits"]))
        return {k: state[k] for k in ("experts", "weights", "offsets", "slots", "dlogits")}
    if case["gradient"]:
        plan.Backward(_at(state["dout"]), _at(state["y"]), _at(state["slots"]), _at(state["weights"]), _at(state["dy"]), _at(state["dweights"]))
        return {"dy": state["dy"], "dweights": state["dweights"]}
    plan.Run(_at(state["y"]), _at(state["slots"]), _at(state["weights"]), _at(state["out"]))
    return {"out": state["out"]}


def _loads(E, M, gen):
    """Rows of each of E experts, M in all, as a router that has favourites gives them; the second expert has none."""
    share = torch.exp(torch.randn(E, device="cuda", generator=gen) * 0.7)
    share[1] = 0.0
    counts = torch.bincount(torch.multinomial(share, M, replacement=True, generator=gen), minlength=E)
    return torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)


def _slots(T, k, gen):
    """Places of k rows of each of T tokens: what sorting them by one of 64 experts gives."""
    experts = torch.rand((T, 64), device="cuda", generator=gen).argsort(dim=1)[:, :k].flatten()
    order = torch.argsort(experts, stable=True)
    slots = torch.empty_like(order)
    slots[order] = torch.arange(T * k, device="cuda")
    return slots.view(T, k).to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    path, t = case["path"], TORCH[case["t"]]
    state = {"case": dict(case)}

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, device="cuda", generator=gen) * scale).to(t)

    def empty(*shape, dtype=t):
        return torch.empty(shape, dtype=dtype, device="cuda")

    if path in ("linear", "grouped", "linear_gradient", "grouped_gradient"):
        M, N, K = case["M"], case["N"], case["K"]
        experts = (case["E"],) if path.startswith("grouped") else ()
        state["x"] = _activations((M, K), gen).to(t)
        state["w"] = normal(*experts, N, K, scale=K ** -0.5)
        if experts:
            state["offsets"] = _loads(case["E"], M, gen)
            state["starts"] = state["offsets"].tolist()
        if path.endswith("gradient"):
            g = TORCH[case["tgrad"]]
            state["dy"], state["z"] = _gradients((M, N), gen).to(t), normal(M, N)
            state["dx"] = empty(M, K)
            state["dw"], state["db"] = empty(*experts, N, K, dtype=g), empty(*experts, N, dtype=g)
            if case["accumulate"]:
                state["dw"].copy_(normal(N, K))
                state["db"].copy_(normal(N))
        else:
            state["b"] = normal(*experts, N, scale=0.5) if case["bias"] else None
            state["r"] = normal(M, N) if case.get("residual") else None
            state["y"], state["z"] = empty(M, N), empty(M, N) if case.get("keep") else None
    elif path == "route":
        T, E, k = case["T"], case["E"], case["k"]
        state["logits"] = (torch.randn((T, E), device="cuda", generator=gen) * 2.0
                           + torch.randn(E, device="cuda", generator=gen)).to(t)
        state["dweights"] = torch.randn((T, k), device="cuda", generator=gen) * 1e-2
        state["experts"], state["slots"] = empty(T, k, dtype=torch.int32), empty(T, k, dtype=torch.int32)
        state["weights"], state["offsets"] = empty(T, k, dtype=torch.float32), empty(E + 1, dtype=torch.int32)
        state["dlogits"] = empty(T, E)
    else:
        T, k, N = case["T"], case["k"], case["N"]
        state["y"], state["slots"] = normal(T * k, N), _slots(T, k, gen)
        w = torch.exp(torch.randn((T, k), device="cuda", generator=gen))
        state["weights"] = w / w.sum(dim=1, keepdim=True)
        state["out"] = empty(T, N)
        if case["gradient"]:
            state["dout"] = _gradients((T, N), gen).to(t)
            state["dy"], state["dweights"] = empty(T * k, N), empty(T, k, dtype=torch.float32)
    return state


def run(state):
    return _own(state) if own else _plain(state)


def _asked(E, rows):
    """How many of E experts `rows` rows go to, about."""
    return min(E, max(1, round(E * (1.0 - (1.0 - 1.0 / E) ** rows))))


def work(case):
    path, size = case["path"], BYTES[case["t"]]
    if path in ("linear", "grouped", "linear_gradient", "grouped_gradient"):
        M, N, K = case["M"], case["N"], case["K"]
        E = _asked(case["E"], M) if path.startswith("grouped") else 1
        if path.endswith("gradient"):
            # dy, z (where there is an activation), x and W come in, dx goes out, and dW and db in their own type
            grad = BYTES[case["tgrad"]] * (2 if case["accumulate"] else 1)
            kept = 0 if case["activation"] == "none" else M * N
            experts = case.get("E", 1)
            return {"bytes": size * (M * N + kept + 2 * M * K + E * N * K) + grad * experts * N * (K + 1),
                    "flops": 4 * M * N * K}
        outs = 1 + (1 if case.get("residual") else 0) + (1 if case.get("keep") else 0)
        return {"bytes": size * (M * K + E * N * (K + (1 if case["bias"] else 0)) + outs * M * N), "flops": 2 * M * N * K}
    if path == "route":
        T, E, k = case["T"], case["E"], case["k"]
        return {"bytes": 2 * size * T * E + 16 * T * k + 4 * (E + 1), "flops": 0}
    T, k, N = case["T"], case["k"], case["N"]
    if case["gradient"]:
        return {"bytes": size * (2 * T * k * N + T * N) + 12 * T * k, "flops": 0}
    return {"bytes": size * (T * k * N + T * N) + 8 * T * k, "flops": 0}


# ---- 64 bits -------------------------------------------------------------------------------------------------------

def _act_64(z, activation):
    """act(z) and act'(z)"""
    if activation == "relu":
        return z.clamp(min=0.0), (z > 0).double()
    if activation == "gelu":
        a = math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3)
        inner = math.sqrt(2.0 / math.pi) * (1.0 + 3 * 0.044715 * z ** 2)
        return 0.5 * z * (1.0 + torch.tanh(a)), 0.5 * (1.0 + torch.tanh(a)) + 0.5 * z * inner / torch.cosh(a.clamp(-300, 300)) ** 2
    if activation == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * torch.sigmoid(-z)
    return z, torch.ones_like(z)


def exact(case, seed):
    """What run() returns for these inputs, in 64 bits."""
    state = prepare(case, seed)
    path = case["path"]
    if path in ("linear", "grouped", "linear_gradient", "grouped_gradient"):
        M, N, K = case["M"], case["N"], case["K"]
        if path.startswith("grouped"):
            starts, ws = state["starts"], state["w"]
        else:
            starts, ws = [0, M], state["w"][None]

        def zeros(*shape):
            return torch.zeros(shape, dtype=torch.float64, device="cuda")
        if path.endswith("gradient"):
            out = {"dx": zeros(M, K), "dw": zeros(len(ws), N, K), "db": zeros(len(ws), N)}
        else:
            out = {"y": zeros(M, N), "z": zeros(M, N)}
        for e, w in enumerate(ws):
            rows = slice(starts[e], starts[e + 1])
            x, w = state["x"][rows].double(), w.double()
            if path.endswith("gradient"):
                dz = state["dy"][rows].double() * _act_64(state["z"][rows].double(), case["activation"])[1]
                out["dx"][rows] = torch.mm(dz, w)
                out["dw"][e] = torch.mm(dz.t().contiguous(), x)
                out["db"][e] = dz.sum(dim=0)
            else:
                z = torch.mm(x, w.t().contiguous())
                if state["b"] is not None:
                    z += (state["b"][e] if path == "grouped" else state["b"]).double()
                out["z"][rows], out["y"][rows] = z, _act_64(z, case["activation"])[0]
        if path == "linear" and state["r"] is not None:
            out["y"] += state["r"].double()
        if not path.endswith("gradient"):
            return out if case.get("keep") else {"y": out["y"]}
        if path == "linear_gradient":
            out["dw"], out["db"] = out["dw"][0], out["db"][0]
            if case["accumulate"]:
                out["dw"], out["db"] = out["dw"] + state["dw"].double(), out["db"] + state["db"].double()
        return out
    if path == "route":
        logits, k, E = state["logits"].double(), case["k"], case["E"]
        experts = torch.sort(-logits, dim=1, stable=True)[1][:, :k]
        chosen = torch.zeros_like(logits, dtype=torch.bool).scatter_(1, experts, True)
        p = torch.softmax(logits.masked_fill(~chosen, -math.inf) if case["normalize"] else logits, dim=1)
        weights, dw = p.gather(1, experts), state["dweights"].double()
        spread = torch.zeros_like(logits).scatter_(1, experts, dw)
        flat = experts.flatten().tolist()
        places, at = sorted(range(len(flat)), key=flat.__getitem__), [0] * len(flat)
        for place, row in enumerate(places):
            at[row] = place
        counts = torch.bincount(experts.flatten(), minlength=E)
        return {"experts": experts.to(torch.int32), "weights": weights,
                "offsets": torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32),
                "slots": torch.tensor(at, dtype=torch.int32, device="cuda").view(-1, k),
                "dlogits": p * (spread - (weights * dw).sum(dim=1, keepdim=True))}
    y, slots, weights = state["y"].double(), state["slots"].long(), state["weights"].double()
    T, k = slots.shape
    if case["gradient"]:
        d, dy = state["dout"].double(), torch.zeros_like(y)
        dweights = torch.zeros_like(weights)
        for j in range(k):
            dy[slots[:, j]] = weights[:, j:j + 1] * d
            dweights[:, j] = (y[slots[:, j]] * d).sum(dim=1)
        return {"dy": dy, "dweights": dweights}
    out = torch.zeros((T, y.shape[1]), dtype=torch.float64, device="cuda")
    for j in range(k):
        out += weights[:, j:j + 1] * y[slots[:, j]]
    return {"out": out}
