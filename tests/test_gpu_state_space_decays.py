"""Linear attention with decays where single tokens wipe the state: time steps of thousands, beside each other and in front of small ones."""
import pytest
import torch

from tests.test_gpu_state_space import Problem, check_scan, ints, on_gpu, within

pytestmark = pytest.mark.gpu

WHERE = {"apart": [3, 64, 100, 150], "in_front": list(range(50)) + list(range(64, 70)), "every": list(range(192))}


def problem(step, where, rate):
    # (outputs of up to some step * 4 * size^3 stay within fp16)
    pr = Problem([192], 2, 1, 8, 16, seed=15, starts=[2], size=0.3)
    pr.a[:] = torch.tensor([-rate, -0.9 * rate])
    pr.dt_bias[:] = 0.0
    pr.dt[:] = -5.0
    shares = 0.9 + 0.1 * torch.rand(192, 2, generator=torch.Generator().manual_seed(2))
    pr.dt[WHERE[where]] = (step * shares)[WHERE[where]].half()
    return pr


@pytest.mark.parametrize("step", [1000.0, 4000.0, 60000.0])
@pytest.mark.parametrize("where", WHERE)
@pytest.mark.parametrize("rate", [1.0, 16.0, 1000.0, 1e30])
def test_prompts(gpu, step, where, rate):
    check_scan(problem(step, where, rate), gpu)


@pytest.mark.parametrize("step", [1000.0, 60000.0])
def test_rows_of_a_prompt_are_what_single_tokens_are(gpu, step):
    """every token wipes what was before it, so that each is the same as a request of its own"""
    from uniql_amd import ops
    pr = problem(step, "every", 16.0)
    y, tol, _, _ = pr.want_scan()
    args = [on_gpu(t, gpu) for t in (pr.x, pr.dt)] + [pr.a.to(gpu)] + [on_gpu(t, gpu) for t in (pr.b, pr.c)]
    more = dict(d=pr.d.to(gpu), dt_bias=pr.dt_bias.to(gpu))
    prompt = ops.state_space_scan(*args, cu=ints(pr.cu, gpu), **more)
    single = ops.state_space_scan(*args, state=torch.zeros(192, 2, 8, 16, device=gpu), **more)
    within(prompt, y, tol), within(single, y, tol)
    within(prompt, single.cpu().double(), 2 * tol)
