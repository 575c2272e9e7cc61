"""Linear attention with decays over heads of odd width that lie at even distances: the last channel of a chunk's last row is as good as the others,
and what lies behind it belongs to nobody."""
import pytest
import torch

from tests.test_gpu_state_space import Problem, ints, on_gpu, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,p,n,head", [(2, 53, 96, 54), (2, 53, 96, 64), (1, 27, 128, 28), (2, 65, 64, 66), (1, 127, 256, 128), (3, 1, 8, 2), (4, 63, 128, 64)])
@pytest.mark.parametrize("lengths", [[64], [128, 5], [37, 1, 64, 3], [1000]])
def test_odd_widths_at_even_distances(gpu, heads, p, n, head, lengths):
    from uniql_amd import ops
    pr = Problem(lengths, heads, 1, p, n, seed=p, shift=(heads * p + heads) % 2)
    rows = pr.rows
    # x ends with its last value; each row's heads are `head` apart, with NaN between them
    numbers = (rows * heads - 1) * head + p
    buf = torch.full((numbers,), float("nan"), dtype=torch.float16)
    x = buf.as_strided((rows, heads, p), (heads * head, head, 1))
    x.copy_(pr.x)
    x[:, :, -1] = 3.0
    pr.x = x
    b, c = (torch.empty(rows, 1, n, dtype=torch.float16).copy_(t) for t in (pr.b, pr.c))
    pr.b, pr.c = b, c
    y, tol, S, S_tol = pr.want_scan()
    state = pr.state.to(gpu)
    on_device = buf.to(gpu).as_strided(x.shape, x.stride())
    out = torch.full((rows, heads, head), 7.0, dtype=torch.float16, device=gpu)[:, :, :p]
    got = ops.state_space_scan(on_device, on_gpu(pr.dt, gpu), pr.a.to(gpu), b.to(gpu), c.to(gpu), d=pr.d.to(gpu), dt_bias=pr.dt_bias.to(gpu), state=state,
                               cu=ints(pr.cu, gpu), places=ints(pr.places, gpu), starts=ints(pr.starts, gpu), out=out)
    within(got, y, tol)
    within(state, S, S_tol)
    if head > p:
        assert (out.as_strided((rows, heads, head - p), (heads * head, head, 1), out.storage_offset() + p) == 7.0).all()
