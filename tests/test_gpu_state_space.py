"""What stands between the projections of a state-space layer - causal convolution, linear attention with decays, gated norm - against
64-bit arithmetic."""
import math

import pytest
import torch

from tests import state_space_reference as R

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


def on_gpu(t, dev):
    """a copy on the device that lies as t does"""
    if t is None:
        return None
    base = t._base if t._base is not None else t
    return base.to(dev).as_strided(t.size(), t.stride(), t.storage_offset())


def ints(values, dev):
    return None if values is None else torch.tensor(values, dtype=torch.int32, device=dev)


def within(got, want, tol, what=""):
    got = got.cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    # fp16 rounds what reaches 65520 to infinity: right where the value may lie there
    beyond = torch.isinf(got) & (want.abs() + tol >= 65520.0) & (got.sign() == want.sign())
    off = torch.where(beyond, torch.zeros_like(want), (got - want).abs() - tol)
    assert (off <= 0).all(), (what, float(off.max()), int((~(off <= 0)).sum()))


class Problem:
    """Sequences of `lengths` rows behind each other, `first` rows in front and `behind` rows after them.  Rows of x | b | c and of dt are
    ranges of a wider buffer, `shift` elements into it.  starts: every second sequence is continued, or as given."""

    def __init__(self, lengths, heads=2, groups=1, p=8, n=16, width=4, seed=0, first=0, behind=0, shift=0, starts="mixed", decay=4.0, spare=2,
                 size=1.0):
        gen = torch.Generator().manual_seed(seed * 1000 + len(lengths))
        self.lengths, self.cu = lengths, R.offsets(lengths, first)
        self.count, self.rows = len(lengths), self.cu[-1] + behind
        self.heads, self.groups, self.p, self.n = heads, groups, p, n
        inner, channels = heads * p, heads * p + 2 * groups * n
        self.channels = channels
        pitch = channels + heads + shift
        buf = (torch.randn(self.rows * pitch + shift, generator=gen) * size).half()
        rows = buf[shift:].view(self.rows, pitch)
        self.mixed, self.dt = rows[:, :channels], rows[:, channels:channels + heads]
        self.x = rows[:, :inner].view(self.rows, heads, p)
        self.b = rows[:, inner:inner + groups * n].view(self.rows, groups, n)
        self.c = rows[:, inner + groups * n:channels].view(self.rows, groups, n)
        self.a = -decay * torch.rand(heads, generator=gen) - 0.05
        self.d, self.dt_bias = torch.randn(heads, generator=gen), torch.randn(heads, generator=gen) - 2.0
        self.places = torch.randperm(self.count + spare, generator=gen)[:self.count].tolist()
        self.starts = [5 * (s % 2) for s in range(self.count)] if starts == "mixed" else starts
        self.state = torch.randn(self.count + spare, heads, p, n, generator=gen)
        self.weight = torch.randn(channels, width, generator=gen).half()
        self.bias = torch.randn(channels, generator=gen).half()
        self.conv_state = torch.randn(self.count + spare, width - 1, channels, generator=gen).half()

    def sequences(self):
        for s in range(self.count):
            yield s, slice(self.cu[s], self.cu[s + 1]), self.places[s], self.starts is None or self.starts[s] > 0

    def want_scan(self, d=True, bias=True, **kw):
        y = torch.full((self.rows, self.heads, self.p), NAN, dtype=torch.float64)
        tol = torch.zeros_like(y)
        S, S_tol = self.state.double().clone(), torch.zeros_like(self.state, dtype=torch.float64)
        for _, rows, place, continued in self.sequences():
            if place < 0 or rows.start == rows.stop:
                continue
            old = self.state[place] if continued else torch.zeros_like(self.state[place])
            y[rows], tol[rows], S[place], S_tol[place] = R.scan(self.x[rows], self.dt[rows], self.a, self.b[rows], self.c[rows], self.d if d else None,
                                                               self.dt_bias if bias else None, old, **kw)
        return y, tol, S, S_tol

    def want_conv(self, activation=True, bias=True):
        y = torch.full((self.rows, self.channels), NAN, dtype=torch.float64)
        tol, S = torch.zeros_like(y), self.conv_state.double().clone()
        for _, rows, place, continued in self.sequences():
            if place < 0 or rows.start == rows.stop:
                continue
            old = self.conv_state[place] if continued else torch.zeros_like(self.conv_state[place])
            y[rows], tol[rows], S[place] = R.conv(self.mixed[rows], self.weight, self.bias if bias else None, old, activation)
        return y, tol, S

    def covered(self):
        rows = torch.zeros(self.rows, dtype=torch.bool)
        for _, r, place, _ in self.sequences():
            if place >= 0:
                rows[r] = True
        return rows


def run_scan(pr, dev, d=True, bias=True, in_place=True, cu=True, **kw):
    from uniql_amd import ops
    state = pr.state.to(dev)
    out = torch.full((pr.rows, pr.heads, pr.p), 7.0, dtype=torch.float16, device=dev)
    state_out = None if in_place else state.clone()
    before = state.clone()
    y = ops.state_space_scan(on_gpu(pr.x, dev), on_gpu(pr.dt, dev), pr.a.to(dev), on_gpu(pr.b, dev), on_gpu(pr.c, dev),
                             d=pr.d.to(dev) if d else None, dt_bias=pr.dt_bias.to(dev) if bias else None, state=state,
                             cu=ints(pr.cu, dev) if cu else None, places=ints(pr.places, dev), starts=ints(pr.starts, dev), state_out=state_out,
                             out=out, **kw)
    assert y.data_ptr() == out.data_ptr()
    if not in_place:
        assert torch.equal(state.view(torch.int32), before.view(torch.int32))
    return y, state if in_place else state_out


def check_scan(pr, dev, want=None, **kw):
    wants = {k: v for k, v in kw.items() if k in ("d", "bias", "softplus")}
    if "dt_limit" in kw:
        wants["limit"] = kw["dt_limit"]
    y, tol, S, S_tol = want or pr.want_scan(**wants)
    got, state = run_scan(pr, dev, **kw)
    rows = pr.covered()
    within(got[rows.to(dev)], y[rows], tol[rows], "y")
    assert (got[~rows.to(dev)] == 7.0).all()
    within(state, S, S_tol, "state")


def run_conv(pr, dev, in_place=True, cu=True, activation=True, bias=True):
    from uniql_amd import ops
    state = pr.conv_state.to(dev)
    out = torch.full((pr.rows, pr.channels), 7.0, dtype=torch.float16, device=dev)
    state_out = None if in_place else state.clone()
    y = ops.causal_conv(on_gpu(pr.mixed, dev), pr.weight.to(dev), pr.bias.to(dev) if bias else None, state=state, cu=ints(pr.cu, dev) if cu else None,
                        places=ints(pr.places, dev), starts=ints(pr.starts, dev), state_out=state_out, activation=activation, out=out)
    return y, state if in_place else state_out


def check_conv(pr, dev, **kw):
    y, tol, S = pr.want_conv(**{k: v for k, v in kw.items() if k in ("activation", "bias")})
    got, state = run_conv(pr, dev, **kw)
    rows = pr.covered()
    within(got[rows.to(dev)], y[rows], tol[rows], "y")
    assert (got[~rows.to(dev)] == 7.0).all()
    within(state, S, torch.zeros_like(S), "state")


LENGTHS = [[1], [1, 1, 1], [2, 0, 3, 1], [3], [31, 32, 33], [63, 64, 65], [0, 0, 200, 0], [129, 1, 5, 70]]


# ---- convolution --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("width,p,n,shift", [(4, 8, 16, 0), (3, 7, 5, 1), (2, 33, 1, 3)])
def test_conv(gpu, lengths, width, p, n, shift):
    check_conv(Problem(lengths, p=p, n=n, width=width, seed=width + shift, shift=shift, first=2, behind=3), gpu)


def test_conv_wide_and_without_extras(gpu):
    pr = Problem([40, 7, 90], heads=40, groups=2, p=54, n=96, seed=3)
    check_conv(pr, gpu)
    check_conv(pr, gpu, activation=False, bias=False, in_place=False)


def test_conv_of_single_tokens(gpu):
    pr = Problem([1] * 9, heads=16, p=64, n=64, starts=None, seed=4)
    check_conv(pr, gpu, cu=False)
    pr.places[3] = -1
    check_conv(pr, gpu, cu=False)
    pr.starts = [0, 1, 0, 1, 1, 0, 1, 1, 1]
    check_conv(pr, gpu, cu=False)


def test_conv_many_sequences(gpu):
    """more sequences than a wave looks at in one go, empty ones among them"""
    gen = torch.Generator().manual_seed(5)
    lengths = torch.randint(0, 6, (300,), generator=gen).tolist()
    lengths[60:140] = [0] * 80
    pr = Problem(lengths, p=4, n=4, seed=6, first=1, behind=40)
    pr.places[7], pr.places[150] = -1, pr.count + 100
    check = pr.places[150]
    pr.places[150] = -1
    y, tol, S = pr.want_conv()
    rows = pr.covered()
    pr.places[150] = check   # behind the pool: left out likewise
    got, state = run_conv(pr, gpu)
    within(got[rows.to(gpu)], y[rows], tol[rows])
    assert (got[~rows.to(gpu)] == 7.0).all()
    within(state, S, torch.zeros_like(S))


def test_conv_does_not_look_across_sequences(gpu):
    """infinities and NaN in other sequences, in rows outside and in states of sequences that begin"""
    pr = Problem([5, 40, 2, 37], seed=7, first=1, behind=2, starts=[0, 0, 3, 0])
    pr.mixed[0], pr.mixed[-2:] = NAN, INF
    pr.mixed[pr.cu[0]:pr.cu[1]] = NAN
    pr.mixed[pr.cu[2]:pr.cu[3]] = INF
    for s in (1, 3):
        pr.conv_state[pr.places[s]] = NAN
    y, tol, _ = pr.want_conv()
    got, _ = run_conv(pr, gpu)
    for s in (1, 3):
        rows = slice(pr.cu[s], pr.cu[s + 1])
        within(got[rows], y[rows], tol[rows])


# ---- scan ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("heads,groups,p,n,shift", [(2, 1, 8, 16, 0), (4, 2, 64, 128, 0), (3, 3, 7, 5, 1), (2, 1, 54, 96, 2)])
def test_scan(gpu, lengths, heads, groups, p, n, shift):
    check_scan(Problem(lengths, heads, groups, p, n, seed=p + n, shift=shift, first=2, behind=3), gpu)


@pytest.mark.parametrize("heads,groups,p,n", [(1, 1, 1, 1), (2, 1, 128, 16), (8, 1, 64, 256), (2, 2, 65, 33), (1, 1, 16, 160), (2, 1, 100, 250),
                                              (16, 2, 42, 80), (2, 1, 32, 64)])
def test_scan_sizes(gpu, heads, groups, p, n):
    check_scan(Problem([70, 3, 130], heads, groups, p, n, seed=p), gpu)


@pytest.mark.parametrize("lengths", [[1000], [300, 700], [5, 900, 64, 1, 0, 400], [128] * 6])
@pytest.mark.parametrize("in_place", [True, False])
def test_scan_over_segments(gpu, lengths, in_place):
    """few heads: the workgroups share a sequence's chunks out and put its state together"""
    check_scan(Problem(lengths, 2, 1, 12, 24, seed=sum(lengths), decay=0.3), gpu, in_place=in_place)


def test_scan_many_sequences(gpu):
    gen = torch.Generator().manual_seed(8)
    lengths = torch.randint(0, 9, (300,), generator=gen).tolist()
    lengths[60:140] = [0] * 80
    lengths[200] = 150
    pr = Problem(lengths, 2, 1, 6, 8, seed=9, first=1, behind=40)
    pr.places[7] = pr.places[201] = -1
    check_scan(pr, gpu)


def test_scan_without_extras_and_with_limits(gpu):
    pr = Problem([90, 4, 33], 2, 1, 16, 32, seed=10)
    check_scan(pr, gpu, d=False, bias=False)
    check_scan(pr, gpu, dt_limit=(0.05, 0.2))
    check_scan(pr, gpu, softplus=False, dt_limit=(0.0, 0.5))


@pytest.mark.parametrize("cu", [True, False])
@pytest.mark.parametrize("heads,groups,p,n", [(2, 1, 8, 16), (4, 2, 64, 128), (2, 1, 54, 96), (3, 1, 7, 5), (2, 2, 128, 256), (2, 1, 65, 130), (5, 1, 1, 1),
                                              (2, 1, 30, 32), (2, 1, 64, 64), (1, 1, 100, 255)])
def test_single_tokens(gpu, cu, heads, groups, p, n):
    """with and without offsets"""
    pr = Problem([1] * 7, heads, groups, p, n, seed=n, starts=None)
    pr.places[2] = -1
    check_scan(pr, gpu, cu=cu)
    pr.starts = [0, 1, 0, 4, 1, 0, 2]
    for s in (0, 5):
        pr.state[pr.places[s]] = NAN   # not looked at
    y, tol, S, S_tol = pr.want_scan()
    check_scan(pr, gpu, cu=cu, in_place=False, want=(y, tol, S, S_tol))
    check_scan(pr, gpu, cu=cu, want=(y, tol, S, S_tol), dt_limit=(0.0, INF))


def test_scan_without_states(gpu):
    """every sequence begins with an empty state, and the new ones are dropped or kept"""
    from uniql_amd import ops
    pr = Problem([70, 0, 5, 200], 2, 1, 16, 32, seed=11, starts=[0] * 4)
    y, tol, S, S_tol = pr.want_scan()
    args = [on_gpu(t, gpu) for t in (pr.x, pr.dt)] + [pr.a.to(gpu)] + [on_gpu(t, gpu) for t in (pr.b, pr.c)]
    more = dict(d=pr.d.to(gpu), dt_bias=pr.dt_bias.to(gpu), cu=ints(pr.cu, gpu))
    within(ops.state_space_scan(*args, **more), y, tol)
    within(ops.state_space_scan(*args, places=ints([3, 0, 1 << 30, 5], gpu), **more), y, tol)
    state = pr.state.to(gpu)
    within(ops.state_space_scan(*args, places=ints(pr.places, gpu), state_out=state, **more), y, tol)
    within(state, S, S_tol)
    whole = ops.causal_conv(on_gpu(pr.mixed, gpu), pr.weight.to(gpu), pr.bias.to(gpu), cu=ints(pr.cu, gpu))
    want, tol, _ = pr.want_conv()
    within(whole, want, tol)


def test_scan_does_not_look_across_sequences(gpu):
    pr = Problem([5, 140, 2, 70], 2, 1, 16, 32, seed=12, first=1, behind=2, starts=[0, 0, 3, 0])
    for t in (pr.mixed, pr.dt):
        t[0], t[-2:] = NAN, INF
        t[pr.cu[0]:pr.cu[1]] = NAN
        t[pr.cu[2]:pr.cu[3]] = INF
    for s in (1, 3):
        pr.state[pr.places[s]] = NAN
    y, tol, S, S_tol = pr.want_scan()
    got, state = run_scan(pr, gpu)
    for s in (1, 3):
        rows = slice(pr.cu[s], pr.cu[s + 1])
        within(got[rows], y[rows], tol[rows])
        within(state[pr.places[s]], S[pr.places[s]], S_tol[pr.places[s]])


@pytest.mark.parametrize("what", ["x", "b", "c", "dt"])
@pytest.mark.parametrize("value", [NAN, INF, -INF])
@pytest.mark.parametrize("at", [0, 40, 63, 64, 100])
def test_scan_rows_do_not_see_later_ones(gpu, what, value, at):
    """a value that is no number in one row: the rows in front of it are as without it, and so are, for x, the other channels throughout"""
    pr = Problem([200], 2, 1, 16, 32, seed=13, starts=[0])
    clean, tol, S, S_tol = pr.want_scan()
    if what == "x":
        pr.x[at, 1, 3] = value
    elif what == "dt":
        pr.dt[at, 1] = value
    else:
        getattr(pr, what)[at, 0, 7] = value
    got, state = run_scan(pr, gpu)
    within(got[:at], clean[:at], tol[:at])
    if what == "x":
        others = [i for i in range(32) if i != 19]
        within(got.flatten(1)[:, others], clean.flatten(1)[:, others], tol.flatten(1)[:, others])
        within(state[pr.places[0]].flatten(0, 1)[others], S[pr.places[0]].flatten(0, 1)[others], S_tol[pr.places[0]].flatten(0, 1)[others])
        assert not torch.isfinite(got[at:, 1, 3]).any()
    elif what == "c":
        others = [i for i in range(200) if i != at]
        within(got[others], clean[others], tol[others])
        within(state, S, S_tol)
        assert not torch.isfinite(got[at]).any()
    elif what == "b":
        assert not torch.isfinite(got[at]).any()
    elif value != -INF:   # minus infinity is a time step of 0
        within(got[:, 0], clean[:, 0], tol[:, 0])
        assert not torch.isfinite(got[at:, 1]).any()


@pytest.mark.parametrize("size", [1e-3, 30.0])
def test_scan_of_large_and_small_values(gpu, size):
    """weights and states beyond fp16's range, and far below its smallest number"""
    pr = Problem([150, 64], 2, 1, 16, 64, seed=14, size=size, decay=0.1)
    pr.dt[:] = torch.randn(pr.dt.shape, generator=torch.Generator().manual_seed(1)).half()
    pr.state *= size ** 2 * 10
    check_scan(pr, gpu)
    check_scan(pr, gpu, d=False)
    pr.dt_bias -= 6.0
    check_scan(pr, gpu, d=False)


def test_scan_behind_a_token_that_wipes_the_state(gpu):
    """time steps of hundreds beside ones of a thousandth: differences of sums keep their digits"""
    pr = Problem([192], 2, 1, 8, 16, seed=15, starts=[2], decay=8.0)
    pr.dt_bias[:] = 0.0
    pr.dt[:] = -5.0
    pr.dt[[3, 64, 100, 150]] = 300.0
    check_scan(pr, gpu)


# ---- norm ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,groups,width,shift", [(1, 1, 1, 0), (3, 2, 8, 0), (5, 8, 1024, 0), (2, 1, 8192, 0), (4, 3, 7, 1), (3, 1, 515, 3), (7, 8, 864, 2),
                                                     (2, 2, 2049, 0), (3, 1, 4096, 5), (2, 1, 20001, 0), (70, 1, 100, 4), (1, 3, 2048, 0)])
def test_norm(gpu, rows, groups, width, shift):
    from uniql_amd import ops
    gen = torch.Generator().manual_seed(width)
    channels = groups * width
    buf = torch.randn(2 * rows * (2 * channels + shift) + shift, generator=gen).half()
    x = buf[:rows * channels].view(rows, channels)
    z = buf[rows * channels + shift:][:rows * (channels + shift)].view(rows, channels + shift)[:, :channels]
    z.mul_(3.0)
    weight = torch.randn(channels, generator=gen).half()
    for eps in (1e-5, 0.1):
        want, tol = R.gated_norm(x, z, weight, groups, eps)
        gx, gz = on_gpu(x, gpu), on_gpu(z, gpu)
        within(ops.gated_group_norm(gx, gz, weight.to(gpu), groups, eps), want, tol)
        within(ops.gated_group_norm(gx, gz, weight.to(gpu), groups, eps, out=gz), want, tol)
        gz = on_gpu(z, gpu)
        within(ops.gated_group_norm(gx, gz, weight.to(gpu), groups, eps, out=gx), want, tol)


def test_norm_of_special_rows(gpu):
    """zeros; values whose squares pass fp16; a NaN stays in its group"""
    from uniql_amd import ops
    x, z = torch.randn(4, 64).half(), torch.full((4, 64), 60000.0).half()
    x[0] = 0
    x[1] = 60000.0
    x[2, 3] = NAN
    z[3] = -60000.0
    want, tol = R.gated_norm(x, z, torch.ones(64).half(), 4, 1e-5)
    got = ops.gated_group_norm(x.to(gpu), z.to(gpu), torch.ones(64).half().to(gpu), 4).cpu().double()
    assert torch.isnan(got[2, :16]).all()
    keep = torch.ones(4, 64, dtype=torch.bool)
    keep[2, :16] = False
    within(got[keep], want[keep], tol[keep])
