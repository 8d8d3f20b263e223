"""Orthogonalize of matrices of zeros: zeros for every epsilon that is not zero, however small; NaN, 0 / 0, for a zero one."""
import pytest
import torch

import ccglib_amd as cc
from scaled_util import WIDE, orthogonalized, stream
from test_orthogonalize_gpu import near, update

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", list(WIDE))
@pytest.mark.parametrize("M,N", [(40, 60), (60, 40), (300, 200), (200, 300)])      # (in one launch, in several)
@pytest.mark.parametrize("epsilon", [1e-7, 1e-21, 1e-22, 1e-30, 2.0 ** -149])
@pytest.mark.parametrize("steps", [1, 5])
def test_zeros_stay_zeros(t, M, N, epsilon, steps):
    g = update(3, M, N, t, torch.Generator().manual_seed(15))
    g[1] = 0
    out = torch.ones_like(g)
    cc.Orthogonalize(3, M, N, 0, stream(), t, steps=steps, epsilon=epsilon).Run(g.data_ptr(), out.data_ptr())
    torch.cuda.synchronize()
    assert not out[1].any()
    assert near(out[[0, 2]], orthogonalized(g[[0, 2]], steps, epsilon=epsilon), t)


@pytest.mark.parametrize("t", list(WIDE))
@pytest.mark.parametrize("M,N", [(40, 60), (300, 200)])
def test_nothing_over_nothing(t, M, N):
    g = update(2, M, N, t, torch.Generator().manual_seed(16))
    g[1] = 0
    out = torch.ones_like(g)
    cc.Orthogonalize(2, M, N, 0, stream(), t, epsilon=0.0).Run(g.data_ptr(), out.data_ptr())
    torch.cuda.synchronize()
    assert bool(torch.isnan(out[1]).all()) and bool(torch.isfinite(out[0]).all())
