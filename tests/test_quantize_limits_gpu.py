"""Quantize where a launch along one axis would hold more work-items than 32 bits count: rows or matrices of one value, whose
scale is |x| / 448 (e4m3) and whose byte is that of 448 with x's sign."""
import pytest
import torch

import ccglib_amd as cc
from scaled_util import stream

pytestmark = pytest.mark.gpu
VT, SG, ST = cc.ValueType, cc.ScaleGroup, cc.ScaleType


def values(count):
    gen = torch.Generator(device="cuda").manual_seed(1)
    return torch.randn((count,), device="cuda", generator=gen, dtype=torch.bfloat16).where(
        torch.rand((count,), device="cuda", generator=gen) > 0.01, torch.zeros((), dtype=torch.bfloat16, device="cuda"))


def check(x, q, scale):
    """x [n], q [n][16], scale [n], a part at a time"""
    for at in range(0, len(x), 2 ** 26):
        v, got = x[at:at + 2 ** 26].float(), q[at:at + 2 ** 26]
        top = torch.full_like(v, 448.0)       # (a division by a tensor is one)
        assert torch.equal(scale[at:at + 2 ** 26], v.abs().clamp(min=2.0 ** -100) / top)
        sign = torch.signbit(v).to(torch.uint8) * 128
        assert torch.equal(got[:, 0], torch.where(v == 0, sign, sign + 0x7e))
        assert not got[:, 1:].any()


def test_rows():
    M = 2 ** 28 + 16                          # (16 rows a block of 256 threads)
    x = values(M)
    q = torch.full((M, 16), 0x55, dtype=torch.uint8, device="cuda")
    s = torch.zeros((1, M), device="cuda")
    cc.Quantize(1, M, 1, 0, stream(), VT.bfloat16).Run(x.data_ptr(), q.data_ptr(), s.data_ptr())
    torch.cuda.synchronize()
    check(x, q, s[0])


@pytest.mark.parametrize("group", list(SG))
@pytest.mark.parametrize("direct", [True, False])
def test_matrices(group, direct):
    B = 2 ** 24 + 24                          # (a block each)
    x = values(B)

    def out():
        return torch.full((B, 16), 0x55, dtype=torch.uint8, device="cuda"), torch.zeros((B, 16), device="cuda")
    (q, s), (qt, st) = out(), out()
    cc.Quantize(B, 1, 1, 0, stream(), VT.bfloat16, group=group).Run(
        x.data_ptr(), q.data_ptr() if direct else 0, s.data_ptr() if direct else 0, qt.data_ptr(), st.data_ptr())
    torch.cuda.synchronize()
    check(x, qt, st[:, 0])
    if direct:
        check(x, q, s[:, 0])


def test_matrices_of_16_rows():
    B, M = 2 ** 24 + 8, 16                    # (16 rows a block, as many matrices as a launch takes and nine more)
    x = values(B * M)
    q, s = torch.full((B * M, 16), 0x55, dtype=torch.uint8, device="cuda"), torch.zeros((B, 1, M), device="cuda")
    cc.Quantize(B, M, 1, 0, stream(), VT.bfloat16).Run(x.data_ptr(), q.data_ptr(), s.data_ptr())
    torch.cuda.synchronize()
    check(x, q, s.view(-1))
