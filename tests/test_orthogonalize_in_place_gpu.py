"""Orthogonalize in place where the rows of the result lie at another distance than those of the updates: a matrix of the result
then lies on others' updates."""
import pytest
import torch

import ccglib_amd as cc
from scaled_util import WIDE, orthogonalized, stream
from test_orthogonalize_gpu import near, update

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", list(WIDE))
@pytest.mark.parametrize("B,M,N", [(1, 60, 100), (40, 60, 100), (300, 96, 64), (7, 33, 33), (5, 260, 131), (3, 131, 300)])
@pytest.mark.parametrize("pitch_in,pitch_out", [(0, 9), (11, 0), (3, 5)])
def test_in_place_with_two_pitches(t, B, M, N, pitch_in, pitch_out):
    pitch_in, pitch_out = N + pitch_in, N + pitch_out
    g = update(B, M, N, t, torch.Generator().manual_seed(17))
    buffer = torch.full((B * M * max(pitch_in, pitch_out) + 16,), 7.0, dtype=WIDE[t], device="cuda")
    of = lambda pitch: buffer[:B * M * pitch].view(B, M, pitch)
    op = cc.Orthogonalize(B, M, N, 0, stream(), t, input_pitch=pitch_in, output_pitch=pitch_out)
    for _ in range(3):      # (the same object again)
        buffer.fill_(7.0)
        of(pitch_in)[:, :, :N] = g
        before = buffer.clone()
        op.Run(buffer.data_ptr(), buffer.data_ptr())
        torch.cuda.synchronize()
        got = of(pitch_out)[:, :, :N].clone()
        assert near(got, orthogonalized(g), t)
        of(pitch_out)[:, :, :N] = before[:B * M * pitch_out].view(B, M, pitch_out)[:, :, :N]
        assert torch.equal(buffer, before), "between the rows of the result, and behind it"


@pytest.mark.parametrize("t", list(WIDE))
def test_the_same_object_out_of_place(t):
    B, M, N = 12, 70, 90
    g = update(B, M, N, t, torch.Generator().manual_seed(18))
    out, want = torch.full((B, M, N + 4), 7.0, dtype=WIDE[t], device="cuda"), torch.empty_like(g)
    cc.Orthogonalize(B, M, N, 0, stream(), t).Run(g.data_ptr(), want.data_ptr())
    cc.Orthogonalize(B, M, N, 0, stream(), t, output_pitch=N + 4).Run(g.data_ptr(), out.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(out[:, :, :N], want) and bool((out[:, :, N:] == 7).all())
