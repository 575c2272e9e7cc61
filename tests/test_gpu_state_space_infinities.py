"""Linear attention with decays behind an infinity in x: its channel is infinite from there on, whatever the number of states."""
import math

import pytest
import torch

from tests.test_gpu_state_space import Problem, run_scan, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("p,n", [(8, 24), (8, 128), (7, 5), (12, 33), (70, 250), (64, 200), (3, 1), (8, 64), (8, 80)])
@pytest.mark.parametrize("lengths", [[200], [1000], [300, 1, 1, 90]])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_channel_stays_infinite(gpu, p, n, lengths, sign):
    """b and c are positive and decays far from 0, so that no sum has infinities of both signs and none fades (d x would have the other
    sign where d < 0, and is left out)"""
    pr = Problem(lengths, 2, 1, p, n, seed=p + n, starts=[0] * len(lengths))
    pr.b.abs_().add_(0.1), pr.c.abs_().add_(0.1)
    pr.a[:] = -0.01
    clean, tol, S, S_tol = pr.want_scan(d=False)
    at = 40
    pr.x[at, 1, 2] = sign * math.inf
    got, state = run_scan(pr, gpu, d=False)
    rows = slice(at, lengths[0])
    assert (got[rows, 1, 2] == sign * math.inf).all(), got[rows, 1, 2]
    assert (state[pr.places[0], 1, 2] == sign * math.inf).all()
    keep = torch.ones(pr.rows, 2, p, dtype=torch.bool)
    keep[rows, 1, 2] = False
    within(got[keep.to(gpu)], clean[keep], tol[keep])
    keep = torch.ones_like(pr.state, dtype=torch.bool)
    keep[pr.places[0], 1, 2] = False
    within(state[keep.to(gpu)], S[keep], S_tol[keep])
