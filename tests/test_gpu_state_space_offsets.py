"""Offsets that fall, or lie outside the call's rows: nothing outside rows and places is written, and what lies outside is cut off."""
import pytest
import torch

from tests.test_gpu_state_space import Problem, ints, on_gpu, within

pytestmark = pytest.mark.gpu

FALLING = [[0, 5, 0, 5, 0, 5], [0, 32, 0, 32, 0, 32], [5, 0, 130, 2, 130], [0, 40, 8, 40, 8, 40, 8, 40], [-3, 70, -(1 << 31), (1 << 31) - 1, 1], [0, 130] * 40]


def guarded(rows, columns, dev, spare=8):
    """an output with rows in front and behind that belong to nobody"""
    whole = torch.full((rows + 2 * spare, columns), 7.0, dtype=torch.float16, device=dev)
    return whole, whole[spare:spare + rows]


def conv(pr, cu, dev, state):
    from uniql_amd import ops
    whole, out = guarded(pr.rows, pr.channels, dev)
    ops.causal_conv(on_gpu(pr.mixed, dev), pr.weight.to(dev), pr.bias.to(dev), state=state, cu=ints(cu, dev), places=ints(pr.places, dev), out=out)
    assert (whole[:8] == 7.0).all() and (whole[-8:] == 7.0).all()
    return out


@pytest.mark.parametrize("cu", FALLING)
def test_conv_of_falling_offsets(gpu, cu):
    rows = min(max(cu), 130)
    pr = Problem([rows] + [0] * (len(cu) - 2), p=8, n=16, seed=len(cu))
    state = pr.conv_state.to(gpu)
    out = conv(pr, cu, gpu, state)
    assert torch.isfinite(out).all()
    others = [p for p in range(state.shape[0]) if p not in pr.places]
    assert torch.equal(state[others].cpu(), pr.conv_state[others])


def test_conv_of_offsets_outside(gpu):
    pr = Problem([5, 0, 33, 40], p=8, n=16, seed=1, starts=None)
    y, tol, S = pr.want_conv()
    for cu in ([-9, 5, 5, 38, 1 << 30], [0, 5, 5, 38, 79], [-(1 << 31), 5, 5, 38, (1 << 31) - 1]):
        state = pr.conv_state.to(gpu)
        within(conv(pr, cu, gpu, state), y, tol)
        within(state, S, torch.zeros_like(S))


def scan(pr, cu, dev, state):
    from uniql_amd import ops
    whole, out = guarded(pr.rows, pr.heads * pr.p, dev)
    ops.state_space_scan(on_gpu(pr.x, dev), on_gpu(pr.dt, dev), pr.a.to(dev), on_gpu(pr.b, dev), on_gpu(pr.c, dev), d=pr.d.to(dev), dt_bias=pr.dt_bias.to(dev),
                         state=state, cu=ints(cu, dev), places=ints(pr.places, dev), out=out.view(pr.rows, pr.heads, pr.p))
    assert (whole[:8] == 7.0).all() and (whole[-8:] == 7.0).all()
    return out.view(pr.rows, pr.heads, pr.p)


@pytest.mark.parametrize("cu", FALLING)
def test_scan_of_falling_offsets(gpu, cu):
    rows = min(max(cu), 130)
    pr = Problem([rows] + [0] * (len(cu) - 2), p=8, n=16, seed=len(cu))
    state = pr.state.to(gpu)
    out = scan(pr, cu, gpu, state)
    assert torch.isfinite(out).all()
    others = [p for p in range(state.shape[0]) if p not in pr.places]
    assert torch.equal(state[others].cpu(), pr.state[others])


def test_a_scan_of_many_more_rows_than_there_are_ends(gpu):
    """10000 sequences of all 6400 rows each are a million chunks for each head: nothing is done"""
    pr = Problem([6400] + [0] * 19998, heads=1, p=8, n=16, seed=2)
    state = pr.state.to(gpu)
    out = scan(pr, [0, 6400] * 10000, gpu, state)
    assert (out == 7.0).all() and torch.equal(state.cpu(), pr.state)


def test_scan_of_offsets_outside(gpu):
    pr = Problem([5, 0, 33, 140], p=8, n=16, seed=1, starts=None)
    y, tol, S, S_tol = pr.want_scan()
    for cu in ([-9, 5, 5, 38, 1 << 30], [0, 5, 5, 38, 179], [-(1 << 31), 5, 5, 38, (1 << 31) - 1]):
        state = pr.state.to(gpu)
        within(scan(pr, cu, gpu, state), y, tol)
        within(state, S, S_tol)
