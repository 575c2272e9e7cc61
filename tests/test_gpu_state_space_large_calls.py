"""Calls of more workgroups than a launch takes: the last rows and sequences are as good as the first."""
import pytest
import torch

from tests import state_space_reference as R
from tests.test_gpu_state_space import within

pytestmark = pytest.mark.gpu


def rows_to_look_at(n):
    gen = torch.Generator().manual_seed(n)
    return torch.cat([torch.arange(5), torch.randint(0, n, (200,), generator=gen), torch.arange(n - 300, n)])


def test_norm(gpu):
    """16500 rows of 4096 groups of 8"""
    from uniql_amd import ops
    rows, groups = 16500, 4096
    gen = torch.Generator(gpu).manual_seed(0)
    x, z = (torch.randn(rows, 8 * groups, generator=gen, device=gpu).half() for _ in range(2))
    weight = torch.randn(8 * groups, generator=gen, device=gpu).half()
    got = ops.gated_group_norm(x, z, weight, groups)
    at = rows_to_look_at(rows)[::8]
    want, tol = R.gated_norm(x[at].cpu(), z[at].cpu(), weight.cpu(), groups, 1e-5)
    within(got[at], want, tol)


def test_steps(gpu):
    """16500 requests of 1024 heads"""
    from uniql_amd import ops
    rows, heads = 16500, 1024
    gen = torch.Generator(gpu).manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=gen, device=gpu)
    x, dt, b, c = r(rows, heads, 1).half(), r(rows, heads).half(), r(rows, 1, 1).half(), r(rows, 1, 1).half()
    a, d, state = -r(heads).abs() - 0.1, r(heads), r(rows, heads, 1, 1)
    before = state.clone()
    got = ops.state_space_scan(x, dt, a, b, c, d=d, state=state)
    for i in rows_to_look_at(rows).tolist()[::16]:
        y, tol, S, S_tol = R.scan(x[i:i + 1].cpu(), dt[i:i + 1].cpu(), a.cpu(), b[i:i + 1].cpu(), c[i:i + 1].cpu(), d.cpu(), None, before[i].cpu())
        within(got[i:i + 1], y, tol), within(state[i], S, S_tol)


def test_convolution(gpu):
    """2^24 requests of 3 channels"""
    from uniql_amd import ops
    rows = 1 << 24
    gen = torch.Generator(gpu).manual_seed(2)
    x, state = torch.randn(rows, 3, generator=gen, device=gpu).half(), torch.randn(rows, 1, 3, generator=gen, device=gpu).half()
    weight, bias = torch.randn(3, 2, generator=gen, device=gpu).half(), torch.randn(3, generator=gen, device=gpu).half()
    before = state.clone()
    got = ops.causal_conv(x, weight, bias, state=state)
    assert torch.equal(state[:, 0], x)
    for i in rows_to_look_at(rows).tolist()[::16]:
        y, tol, _ = R.conv(x[i:i + 1].cpu(), weight.cpu(), bias.cpu(), before[i].cpu())
        within(got[i:i + 1], y, tol)
