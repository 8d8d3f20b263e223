"""Products with nearly as many blocks as a launch takes, and with more than it would take of the smallest blocks: every element
of C is written. The operands' values are one of 1, 2, 4 in the first place of a row and zero behind it, so C is exact."""
import pytest
import torch

import ccglib_amd as cc
from scaled_util import stream

pytestmark = pytest.mark.gpu
VT, SG, ST = cc.ValueType, cc.ScaleGroup, cc.ScaleType


def rows(count, seed):
    """Bytes of `count` rows of 16 e4m3 values, and what the first ones stand for."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    exponent = torch.randint(0, 3, (count,), dtype=torch.uint8, device="cuda", generator=gen)
    held = torch.zeros((count, 16), dtype=torch.uint8, device="cuda")
    held[:, 0] = (exponent + 7) * 8
    return held, exponent


def test_as_many_matrices_as_a_launch_takes():
    B = 2 ** 24 - 1
    a, ea = rows(B, 1)
    b, eb = rows(B, 2)
    scales = torch.ones((B, 1, 16), device="cuda")
    c = torch.zeros((B,), device="cuda")
    op = cc.ScaledGEMM(B, 1, 1, 16, 0, stream(), c_type=VT.float32)
    op.Run(a.data_ptr(), scales.data_ptr(), b.data_ptr(), scales.data_ptr(), c.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(c, torch.exp2((ea + eb).float()))


def test_a_row_of_c_of_2_to_the_30():
    """In blocks of 64 x 32 these would be 2^24."""
    N = 2 ** 30
    a, ea = rows(1, 3)
    b, eb = rows(N, 4)
    one = torch.full((16,), 127, dtype=torch.uint8, device="cuda")
    scales = torch.full((N,), 127, dtype=torch.uint8, device="cuda")
    scales[N - 5:] = 128
    c = torch.zeros((N,), dtype=torch.bfloat16, device="cuda")
    op = cc.ScaledGEMM(1, 1, N, 16, 0, stream(), b_group=SG.rows, scale_type=ST.e8m0)
    op.Run(a.data_ptr(), one.data_ptr(), b.data_ptr(), scales.data_ptr(), c.data_ptr())
    torch.cuda.synchronize()
    eb[N - 5:] += 1
    for at in range(0, N, 2 ** 27):
        assert torch.equal(c[at:at + 2 ** 27].float(), torch.exp2((eb[at:at + 2 ** 27] + ea).float()))
