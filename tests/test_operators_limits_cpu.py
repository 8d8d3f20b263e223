"""Sizes at the upper end of what the operators on real matrices take: what the kernels could not count is refused when an object
is created, before a device is touched; what is just below passes these checks."""
import pytest

import ccglib_amd as cc

VT, SG, ST = cc.ValueType, cc.ScaleGroup, cc.ScaleType


def refusal(make):
    """The error's text; None if there is none, as on a machine with a device."""
    try:
        make()
    except RuntimeError as e:
        return str(e)
    return None


# (32-bit offsets of 4-byte scales: from 2^30 - 15 rows on their row of scales is 2^30 long)
@pytest.mark.parametrize("rows,group,scale,refused", [
    (2 ** 30, SG.rows, ST.float32, True), (2 ** 30 - 15, SG.rows, ST.float32, True), (2 ** 31 - 1, SG.rows, ST.float32, True),
    (2 ** 30 - 16, SG.rows, ST.float32, False), (2 ** 30, SG.rows, ST.e8m0, False), (2 ** 30, SG.blocks, ST.float32, False)])
def test_scales_of_many_rows(rows, group, scale, refused):
    text = refusal(lambda: cc.ScaledGEMM(1, 1, rows, 16, 0, 0, b_group=group, scale_type=scale))
    assert ("4 GiB" in (text or "")) == refused
