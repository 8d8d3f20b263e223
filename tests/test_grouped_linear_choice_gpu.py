"""Which kernel a GroupedLinear's y runs as: that for a few rows reads an expert's W for every 16 of its rows, and the loads are not known
when it is chosen. So it is not, where all rows may go to one expert whose W is read again and again."""
import pytest
import torch

import ccglib_amd as cc
from linear_util import stream

pytestmark = pytest.mark.gpu


def kernel(E, M, N, K):
    return cc.GroupedLinear(E, M, N, K, 0, stream(), training=False).KernelName()


@pytest.mark.parametrize("E,M,N,K", [(128, 256, 8192, 8192), (64, 128, 2048, 2048), (1024, 2048, 1024, 1024), (1024, 64, 512, 512),
                                     (32, 64, 4096, 2048)])
def test_many_rows_of_large_weights(E, M, N, K):
    assert "gemm_linear" in kernel(E, M, N, K)


@pytest.mark.parametrize("E,M,N,K", [(64, 16, 2048, 2048), (8, 1, 8192, 8192), (64, 128, 256, 256), (1024, 16, 512, 512)])
def test_no_more_than_one_block_of_rows_or_little_work(E, M, N, K):
    assert "linear_rows" in kernel(E, M, N, K)


def test_what_is_read_is_bounded_whatever_the_loads():
    """Over the whole range: W's bytes once for each 16 rows, at most 16 rows in all or 1280 blocks whose operands are read once each."""
    for E in (1, 2, 8, 60, 256, 1024):
        for M in (1, 16, 17, 40, 100, 300, 2000):
            for N, K in ((64, 64), (300, 512), (1000, 1024), (2048, 4096), (8192, 8192)):
                if "linear_rows" in kernel(E, M, N, K) and M > 16:
                    assert -(-M // 16) * -(-N // 16) <= 1280 and K <= 5000
    torch.cuda.synchronize()
