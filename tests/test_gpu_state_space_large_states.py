"""Linear attention with decays whose states are large beside what rows add: finite ones stay finite."""
import pytest
import torch

from tests.test_gpu_state_space import Problem, check_scan

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("power", [37, 41, 60, 100, 126])
@pytest.mark.parametrize("dt", [-60000.0, -20.0, 0.0])
@pytest.mark.parametrize("lengths", [[130], [1000], [70, 5, 300]])
def test_states_beside_small_steps(gpu, power, dt, lengths):
    """chunks that add nothing or little; c is zero, since outputs of such states are beyond fp16"""
    pr = Problem(lengths, 2, 1, 8, 24, seed=power, starts=[3] * len(lengths), decay=0.1)
    pr.c[:] = 0.0
    pr.dt_bias[:] = 0.0
    pr.dt[:] = dt
    pr.x[:, 0, :5] = 0.0
    pr.state.clamp_(-1.9, 1.9).mul_(2.0 ** power)
    check_scan(pr, gpu)


def test_a_large_state_and_small_ones(gpu):
    """a state far above the others of its channel leaves them their digits"""
    pr = Problem([200, 1000], 2, 1, 8, 24, seed=3, starts=[3, 3], decay=0.1)
    pr.c[:] = 0.0
    pr.dt[100:164] = -60000.0
    pr.x[64:128, 1, 3] = 0.0
    pr.state[..., 7] = 2.0 ** 60
    check_scan(pr, gpu)


@pytest.mark.parametrize("bias", [1e15, 1e20, 1e25])
def test_large_steps(gpu, bias):
    """time steps beyond fp16, by their bias"""
    pr = Problem([200, 1000], 2, 1, 8, 24, seed=5, starts=[3, 0], decay=0.1)
    pr.c[:] = 0.0
    pr.dt_bias[:] = torch.tensor([bias, 0.3 * bias])
    check_scan(pr, gpu)
    pr.a[:] *= 1.0 / bias
    check_scan(pr, gpu)


@pytest.mark.parametrize("limit", [(0.0, 0.0), (0.0, 1e-30), (1e8, 1e9), (0.0, 3e38)])
def test_limits_of_steps(gpu, limit):
    """none at all, or all longer than fp16 holds"""
    pr = Problem([200, 1000], 2, 1, 8, 24, seed=6, starts=[3, 0], decay=0.1)
    pr.c[:] = 0.0
    pr.state[..., 3] *= 1e12
    pr.a[:] *= 1.0 / max(1.0, limit[0])
    check_scan(pr, gpu, dt_limit=limit)
