"""Quantize: 8-bit values and scales are those of the formula, bit for bit (both are roundings of one number each, so
nothing is tolerated), in both orientations; rows end in zeros."""
import itertools

import pytest
import torch

import ccglib_amd as cc
from scaled_util import F8, WIDE, groups, quantized, scales_64, stream, up

pytestmark = pytest.mark.gpu
VT, SG, ST = cc.ValueType, cc.ScaleGroup, cc.ScaleType

SIZES = [(1, 1, 1), (1, 1, 127), (2, 3, 128), (1, 5, 129), (3, 127, 40), (1, 128, 128), (2, 129, 257), (1, 300, 16), (1, 17, 1000)]


def run(x, B, M, N, vtype, group, scale_type, tin, direct=True, transposed=True, pitch=0, data_ptr=None):
    """Device buffers, filled with 0x55 first: (q, s, qt, st)."""
    dt = torch.uint8 if scale_type == ST.e8m0 else torch.float32

    def out(rows, cols):
        r = rows if group == SG.rows else groups(rows)
        return (torch.full((B, rows, up(cols)), 0x55, dtype=torch.uint8, device="cuda"),
                torch.full((B, groups(cols), up(r)), 77, dtype=dt, device="cuda"))
    q, s = out(M, N)
    qt, st = out(N, M)
    op = cc.Quantize(B, M, N, 0, stream(), tin, vtype, group, scale_type, pitch)
    op.Run(data_ptr or x.data_ptr(), q.data_ptr() if direct else 0, s.data_ptr() if direct else 0,
           qt.data_ptr() if transposed else 0, st.data_ptr() if transposed else 0)
    torch.cuda.synchronize()
    return q, s, qt, st


def check(x, q, s, vtype, group, scale_type):
    B, R, C = x.shape
    want_q, want_s = quantized(x, vtype, group, scale_type)
    got = q[:, :, :C].contiguous().view(F8[vtype][0]).double().cpu()
    assert torch.equal(torch.nan_to_num(got, nan=1e9), torch.nan_to_num(want_q, nan=1e9))
    assert torch.equal(scales_64(s, want_s.shape[2], scale_type), want_s)
    assert not q[:, :, C:].any(), "rows end in zeros"


@pytest.mark.parametrize("tin,vtype", list(itertools.product(WIDE, F8)))
@pytest.mark.parametrize("group,scale_type", list(itertools.product(SG, ST)))
def test_values_and_scales(tin, vtype, group, scale_type):
    gen = torch.Generator().manual_seed(3)
    for B, M, N in SIZES:
        x = torch.randn((B, M, N), generator=gen) * torch.exp(2 * torch.randn((B, M, 1), generator=gen))
        x = x.to(WIDE[tin]).cuda()
        q, s, qt, st = run(x, B, M, N, vtype, group, scale_type, tin)
        check(x, q, s, vtype, group, scale_type)
        check(x.transpose(1, 2), qt, st, vtype, group, scale_type)
        # one orientation alone gives the same, and leaves the other's buffers alone
        q1, s1, qt1, st1 = run(x, B, M, N, vtype, group, scale_type, tin, transposed=False)
        check(x, q1, s1, vtype, group, scale_type)
        assert bool((qt1 == 0x55).all()) and bool((st1 == 77).all())
        q2, s2, qt2, st2 = run(x, B, M, N, vtype, group, scale_type, tin, direct=False)
        check(x.transpose(1, 2), qt2, st2, vtype, group, scale_type)
        assert bool((q2 == 0x55).all()) and bool((s2 == 77).all())


@pytest.mark.parametrize("group,scale_type", list(itertools.product(SG, ST)))
@pytest.mark.parametrize("vtype", list(F8))
@pytest.mark.parametrize("tin", [VT.float32, VT.bfloat16])
def test_zeros_infinities_nan_and_extremes(tin, vtype, group, scale_type):
    """Groups of zeros, of NaN alone, with infinities among ordinary values, near the ends of the type's range."""
    M, N = 260, 400
    gen = torch.Generator().manual_seed(4)
    x = torch.randn((1, M, N), generator=gen)
    x[0, 3] = 0.0
    x[0, 4, :128] = float("nan")
    x[0, 5, 7], x[0, 5, 200], x[0, 6, 11] = float("inf"), float("-inf"), float("nan")
    x[0, 7] *= 1e-38
    x[0, 8] *= 1e37
    x[0, 9] = -0.0
    x[0, 130:260, 130:300] = 0.0           # a whole block, and groups along columns
    x[0, :, 301] = float("inf")
    x = x.to(WIDE[tin]).cuda()
    q, s, qt, st = run(x, 1, M, N, vtype, group, scale_type, tin)
    check(x, q, s, vtype, group, scale_type)
    check(x.transpose(1, 2), qt, st, vtype, group, scale_type)


@pytest.mark.parametrize("vtype", list(F8))
def test_ties_go_to_the_even_neighbour(vtype):
    """The group's largest value is the type's, so the factor is 1; then every midpoint between two neighbours."""
    dtype, top = F8[vtype]
    codes = torch.arange(256, dtype=torch.uint8).view(dtype).float()
    values = torch.sort(codes[torch.isfinite(codes)])[0].unique()
    middle = (values[1:] + values[:-1]) / 2
    x = torch.zeros((1, 1, 3 * 128))
    for g in range(3):
        part = middle[g * 127:(g + 1) * 127]
        x[0, 0, g * 128:g * 128 + len(part)] = part
        x[0, 0, g * 128 + 127] = top
    x = x.cuda()
    q, s, qt, st = run(x, 1, 1, 384, vtype, SG.rows, ST.float32, VT.float32)
    assert bool((s[0, :, 0] == 1).all())
    check(x, q, s, vtype, SG.rows, ST.float32)


@pytest.mark.parametrize("tin", list(WIDE))
@pytest.mark.parametrize("offset", [1, 3])
def test_rows_apart_and_starting_anywhere(tin, offset):
    M, N, pitch = 70, 135, 151
    whole = torch.randn((M * pitch + offset,)).to(WIDE[tin]).cuda()
    x = whole[offset:].view(M, pitch)[None, :, :N]
    for group in SG:
        q, s, qt, st = run(x, 1, M, N, VT.float8e4m3, group, ST.float32, tin, pitch=pitch,
                           data_ptr=whole.data_ptr() + offset * whole.element_size())
        check(x, q, s, VT.float8e4m3, group, ST.float32)
        check(x.transpose(1, 2), qt, st, VT.float8e4m3, group, ST.float32)


def test_empty_matrices_are_left_alone():
    for B, M, N in [(0, 4, 4), (1, 0, 4), (1, 4, 0)]:
        cc.Quantize(B, M, N, 0, stream(), VT.float32).Run(0, 0, 0)


def test_offsets_beyond_32_bits():
    """Rows so far apart that the last one starts past 4 GiB."""
    M, N, pitch = 70000, 40, 32768
    whole = torch.empty((M, pitch), dtype=torch.bfloat16, device="cuda")
    x = torch.randn((1, M, N), device="cuda").to(torch.bfloat16)
    whole[:, :N] = x[0]
    q, s, qt, st = run(None, 1, M, N, VT.float8e4m3, SG.rows, ST.float32, VT.bfloat16, pitch=pitch, data_ptr=whole.data_ptr())
    check(x, q, s, VT.float8e4m3, SG.rows, ST.float32)
    check(x.transpose(1, 2), qt, st, VT.float8e4m3, SG.rows, ST.float32)


def test_refusals_at_run():
    x = torch.zeros(64, device="cuda")
    out = torch.zeros(4096, dtype=torch.uint8, device="cuda")
    op = cc.Quantize(1, 4, 16, 0, stream(), VT.float32)
    with pytest.raises(RuntimeError, match="null pointer: input"):
        op.Run(0, out.data_ptr(), out.data_ptr())
    with pytest.raises(RuntimeError, match="null pointer: output"):
        op.Run(x.data_ptr(), 0, 0)
    with pytest.raises(RuntimeError, match="null pointer"):
        op.Run(x.data_ptr(), out.data_ptr(), 0)
    with pytest.raises(RuntimeError, match="multiple of 16 bytes"):
        op.Run(x.data_ptr(), out.data_ptr() + 8, out.data_ptr())
    with pytest.raises(RuntimeError, match="misaligned scales"):
        op.Run(x.data_ptr(), out.data_ptr(), out.data_ptr() + 2)
    with pytest.raises(RuntimeError, match="misaligned input"):
        op.Run(x.data_ptr() + 2, out.data_ptr(), out.data_ptr())
