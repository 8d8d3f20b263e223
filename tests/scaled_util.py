"""Plain statements, in 64 bits, of the 8-bit operators with block scales and of the orthogonalised updates, and what
their GPU tests share: buffers in the library's layout."""
import torch

import ccglib_amd as cc

GROUP = 128
F8 = {cc.ValueType.float8e4m3: (torch.float8_e4m3fn, 448.0), cc.ValueType.float8e5m2: (torch.float8_e5m2, 57344.0)}
WIDE = {cc.ValueType.float32: torch.float32, cc.ValueType.float16: torch.float16,
        cc.ValueType.bfloat16: torch.bfloat16}


def up(n, to=16):
    return -(-n // to) * to


def groups(n):
    return -(-n // GROUP)


def stream():
    return torch.cuda.current_stream().cuda_stream


def quantized(x, vtype, group, scale_type):
    """(values, scales) in 64 bits, [B][R][C] and [B][C/128][R or R/128], of x [B][R][C]. The scale and the factor are
    numbers of 32 bits; the value times the factor is rounded to 32 bits, then to 8."""
    dtype, top = F8[vtype]
    B, R, C = x.shape
    x = x.double().cpu()
    step = 1 if group == cc.ScaleGroup.rows else GROUP
    rows = -(-R // step)
    padded = torch.zeros((B, rows * step, groups(C) * GROUP), dtype=torch.float64)
    padded[:, :R, :C] = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
    amax = padded.reshape(B, rows, step, groups(C), GROUP).amax(dim=(2, 4)).clamp(min=2.0 ** -100)
    ratio = (amax / top).float().double()          # (a quotient of two numbers of 32 bits, rounded once)
    if scale_type == cc.ScaleType.e8m0:
        mantissa, exponent = torch.frexp(ratio)
        scale = torch.pow(2.0, torch.where(mantissa == 0.5, exponent - 1, exponent).double())
        factor = 1.0 / scale
    else:
        scale, factor = ratio, (top / amax).float().double()
    each = factor.repeat_interleave(step, dim=1)[:, :R].repeat_interleave(GROUP, dim=2)[:, :, :C]
    q = (x * each).float().to(dtype).double()
    return q, scale.transpose(1, 2).contiguous()


def values_of(q, scale, group):
    """What values [B][R][C] with scales [B][C/128][rows] stand for, in 64 bits."""
    step = 1 if group == cc.ScaleGroup.rows else GROUP
    each = scale.transpose(1, 2).repeat_interleave(step, dim=1)[:, :q.shape[1]]
    return q * each.repeat_interleave(GROUP, dim=2)[:, :, :q.shape[2]]


def held(q, scale, vtype, scale_type, pitch=None):
    """Device buffers in the library's layout of values and scales in 64 bits."""
    B, R, C = q.shape
    dtype = F8[vtype][0]
    pitch = pitch or up(C)
    values = torch.zeros((B, R, pitch), dtype=torch.uint8)
    values[:, :, :C] = q.float().to(dtype).view(torch.uint8)
    scales = torch.ones((B, scale.shape[1], up(scale.shape[2])), dtype=torch.float32)
    scales[:, :, :scale.shape[2]] = scale.float()
    if scale_type == cc.ScaleType.e8m0:
        scales = ((scales.view(torch.int32) >> 23) & 0xff).to(torch.uint8)
    return values.cuda(), scales.cuda()


def scales_64(buffer, rows, scale_type):
    """Scales [B][groups][rows] in 64 bits from a buffer of the library's layout."""
    s = buffer[:, :, :rows].cpu()
    return torch.pow(2.0, s.double() - 127.0) if scale_type == cc.ScaleType.e8m0 else s.double()


def random_operand(gen, B, R, C, vtype, group, scale_type, spread=1.0):
    """(values, scales, magnitudes they stand for) of N(0, 1) values whose rows differ in size."""
    x = torch.randn((B, R, C), generator=gen, dtype=torch.float64)
    x = x * torch.exp(spread * torch.randn((B, R, 1), generator=gen, dtype=torch.float64))
    q, s = quantized(x.float(), vtype, group, scale_type)
    return q, s, values_of(q, s, group)


def orthogonalized(g, steps=5, coefficients=(3.4445, -4.7750, 2.0315), epsilon=1e-7):
    a, b, c = (float(torch.tensor(v, dtype=torch.float32)) for v in coefficients)
    out = []
    for x in g.double().cpu():
        x = x / (x.norm() + float(torch.tensor(epsilon, dtype=torch.float32)))
        tall = x.shape[0] > x.shape[1]
        x = x.t().contiguous() if tall else x
        for _ in range(steps):
            s = x @ x.t()
            x = a * x + (b * s + c * (s @ s)) @ x
        out.append(x.t() if tall else x)
    return torch.stack(out)
