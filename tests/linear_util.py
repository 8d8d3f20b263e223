"""Plain statements, in 64 bits, of the 16-bit linear layers and of the routing between experts, how far a result may be
from them, and buffers that lie among NaN."""
import math

import torch

import ccglib_amd as cc

VT, ACT = cc.ValueType, cc.Activation
HALF = {VT.float16: torch.float16, VT.bfloat16: torch.bfloat16}
TORCH = dict(HALF) | {VT.float32: torch.float32}
GELU = math.sqrt(2.0 / math.pi)


def stream():
    return torch.cuda.current_stream().cuda_stream


def half_step(t):
    """The largest error of rounding v to t: half_step * |v|, or half the smallest number above zero."""
    return torch.finfo(t).eps / 2, {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[t]


def rounded(v, t):
    rel, least = half_step(t)
    return rel * v.abs() + least


def argument(z, activation):
    """a with act(z) = z sigmoid(a)"""
    return 2.0 * GELU * (z + 0.044715 * z ** 3) if activation == ACT.gelu else z


def act(z, activation):
    if activation == ACT.none:
        return z
    if activation == ACT.relu:
        return torch.where(z > 0, z, torch.where(z <= 0, torch.zeros_like(z), z))
    return z * torch.sigmoid(argument(z, activation))


def act_gradient(z, activation):
    if activation == ACT.none:
        return torch.ones_like(z)
    if activation == ACT.relu:
        return (z > 0).double()
    a = argument(z, activation)
    slope = 2.0 * GELU * (1.0 + 3 * 0.044715 * z ** 2) if activation == ACT.gelu else torch.ones_like(z)
    s = torch.sigmoid(a)
    return s + z * slope * s * torch.sigmoid(-a)


def act_error(z, activation):
    """Of act evaluated in 32 bits. a is a few roundings off, and so by |a| of them sigmoid(a); the sigmoid takes an exp2, a sum
    and a reciprocal, each a rounding or two of its own: 16 steps of 2^-24 and 4 |a| more, of |act(z)|. Where e^-a overflows,
    the result is 0 and z e^a was meant, less than 1e-34."""
    if activation in (ACT.none, ACT.relu):
        return torch.zeros_like(z)
    return (16 + 4 * argument(z, activation).abs()) * 2.0 ** -24 * act(z, activation).abs() + 1e-34


def act_gradient_error(z, activation):
    """Of act' = s + z a' s (1 - s): as above for both terms, and 2^-23 in 1 - s, which is a difference from 1."""
    if activation in (ACT.none, ACT.relu):
        return torch.zeros_like(z)
    a = argument(z, activation)
    slope = 2.0 * GELU * (1.0 + 3 * 0.044715 * z ** 2) if activation == ACT.gelu else torch.ones_like(z)
    s = torch.sigmoid(a)
    term = (z * slope).abs() * s
    # (where 1 - s has been rounded to 0, e^-a is below 2^-24, and what was left out is no more than term e^-a)
    return (24 + 4 * a.abs()) * 2.0 ** -24 * (s + term * torch.sigmoid(-a)) + 2.0 ** -23 * torch.where(a.abs() < 90, term, 0 * term)


def sum_error(sizes, length):
    """Of sums of `length` products in 32 bits in any order, each addition (at most one a product, and one to join parts of K)
    being off by a last place at most; `sizes`: the sums of the products' magnitudes."""
    return (length + 32) * 2.0 ** -23 * sizes


def forward(x, w, bias, residual, activation):
    """(z, y, error of z, error of y) before rounding to 16 bits, of values in 64 bits."""
    z, size = x @ w.t().contiguous(), x.abs() @ w.abs().t().contiguous()
    if bias is not None:
        z, size = z + bias, size + bias.abs()
    ez = sum_error(size, x.shape[1])
    y, ey = act(z, activation), 1.13 * ez + act_error(z, activation)      # (1.13: the largest slope)
    if residual is not None:
        y = y + residual
        ey = ey + 2.0 ** -23 * (y.abs() + residual.abs())
    return z, y, ez, ey


def backward(dy, z, x, w, activation, t):
    """(dx, dw, db) and their errors before rounding, of values in 64 bits. dz is rounded to t on the way to the products."""
    g = act_gradient(z, activation)
    dz = dy * g
    edb = dy.abs() * act_gradient_error(z, activation) + 2.0 ** -23 * dz.abs()
    edz = edb + rounded(dz, t) if activation != ACT.none else torch.zeros_like(dz)
    dx, dw, db = dz @ w, dz.t().contiguous() @ x, dz.sum(dim=0)
    size = dz.abs() + edz
    edx = edz @ w.abs() + sum_error(size @ w.abs(), w.shape[0])
    edw = edz.t().contiguous() @ x.abs() + sum_error(size.t().contiguous() @ x.abs(), x.shape[0])
    return (dx, dw, db), (edx, edw, edb.sum(dim=0) + sum_error(dz.abs().sum(dim=0), len(dz)))


def check(got, want, error, what=""):
    """Asserts that got (rounded to its type) is no further from want than `error` and the rounding allow."""
    want, error = want.cpu(), error.cpu()
    off = (got.double().cpu() - want).abs() - (error + rounded(want.abs() + error, got.dtype))
    worst = float(torch.nan_to_num(off, nan=math.inf).max()) if off.numel() else 0.0
    assert worst <= 0, "%s: %g more than allowed" % (what, worst)


def among_nan(values, pitch=None, shift=0, before=64):
    """A device tensor that views rows of `values` [R][C] `pitch` apart in a buffer of NaN, starting `shift` elements behind a
    multiple of 16 bytes. What lies around it, and between its rows, is NaN."""
    rows, columns = values.shape
    pitch = pitch or columns
    held = torch.full((before + shift + max(0, rows - 1) * pitch + columns + before,), math.nan, dtype=values.dtype, device="cuda")
    view = held[before + shift:].as_strided((rows, columns), (pitch, 1))
    view.copy_(values)
    return view


def routed(logits, k, normalize):
    """(experts, weights, offsets, slots) of logits [T][E] on the host."""
    T, E = logits.shape
    l = logits.double()
    experts = torch.tensor([sorted(range(E), key=lambda e: (-math.inf if v[e] != v[e] else -v[e], e))[:k] for v in l.tolist()],
                           dtype=torch.int64).reshape(T, k)
    top = l.amax(dim=1, keepdim=True) if T else l[:, :1]
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(l - top)
    chosen = p.gather(1, experts)
    scale = (chosen if normalize else p).sum(dim=1, keepdim=True)
    weights = torch.where(scale == 0, torch.zeros_like(chosen), chosen / scale)
    flat = experts.flatten().tolist()
    slots, counts = [0] * len(flat), [0] * E
    for e in flat:
        counts[e] += 1
    offsets = [sum(counts[:e]) for e in range(E + 1)]
    at = list(offsets)
    for i, e in enumerate(flat):
        slots[i] = at[e]
        at[e] += 1
    return experts, weights, offsets, torch.tensor(slots).reshape(T, k)
