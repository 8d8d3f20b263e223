"""A product has to fit one launch, whose work-items are counted in 32 bits; a layer's three products as well."""
import pytest

import ccglib_amd as cc
from test_operators_limits_cpu import refusal

VT, SG, ST = cc.ValueType, cc.ScaleGroup, cc.ScaleType


# (small matrices: a block of 256 threads each at least, so 2^24 of them are too many; long rows of C: blocks of 128 columns or more)
@pytest.mark.parametrize("B,M,N,refused", [
    (2 ** 24, 16, 16, True), (2 ** 24 + 1, 1, 1, True), (2 ** 25 - 1, 16, 16, True), (2 ** 25 - 1, 1, 40, True),
    (2 ** 24 - 1, 16, 16, False), (1, 1, 2 ** 30, False), (1, 1, 2 ** 31 - 128, False)])
@pytest.mark.parametrize("c_type", [VT.bfloat16, VT.float32])
def test_blocks_of_a_product(B, M, N, refused, c_type):
    text = refusal(lambda: cc.ScaledGEMM(B, M, N, 16, 0, 0, c_type=c_type, scale_type=ST.e8m0))
    assert ("than a launch takes" in (text or "")) == refused


# (64 x 32 blocks of 256 threads: 2^23 of them, K in two parts)
@pytest.mark.parametrize("option,refused", [(4 + 256 * 2, True), (4 + 256, False), (1 + 256 * 2, False), (0, False)])
def test_blocks_of_a_layer(option, refused):
    with cc.option(cc.Option.real_block, option):
        for M, N, K in [(2 ** 22, 2 ** 12, 256), (2 ** 22, 256, 2 ** 12)]:
            text = refusal(lambda: cc.ScaledLinear(M, N, K, 0, 0, training=True))
            assert ("than a launch takes" in (text or "")) == refused
