"""The operators of a state-space layer as they are used: together, in pieces, recorded into graphs, on other streams, far apart in memory;
and what they refuse."""
import pytest
import torch

from tests import state_space_reference as R
from tests.test_gpu_state_space import Problem, check_scan, ints, on_gpu, run_scan, within

pytestmark = pytest.mark.gpu

HEADS, P, GROUPS, N = 4, 12, 2, 24
INNER, CHANNELS = HEADS * P, HEADS * P + 2 * GROUPS * N
WIDTH = INNER + CHANNELS + HEADS


def mixer(dev, seed=0, norm_groups=2, p=P):
    from uniql_amd.state_space import StateSpaceMixer
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    inner, channels = HEADS * p, HEADS * p + 2 * GROUPS * N
    return StateSpaceMixer(HEADS, p, GROUPS, N, r(channels, 1, 4) * 0.5, r(channels) * 0.3, r(HEADS) * 0.5, r(HEADS), r(HEADS) - 2, 1 + 0.2 * r(inner),
                           norm_groups).to(dev)


def projected(rows, dev, seed=1, more=5):
    buf = torch.randn(rows, WIDTH + more, generator=torch.Generator().manual_seed(seed)).half()
    return buf.to(dev)


def in_64_bits(m, h, lengths, conv, ssm, starts):
    """the layer's definition, roundings only where the operators hand over"""
    c = lambda t: None if t is None else t.cpu()
    inner, p = m.num_heads * m.head_dim, m.head_dim
    channels = inner + 2 * GROUPS * N
    h, y = h.cpu(), torch.zeros(sum(lengths), inner, dtype=torch.float64)
    cu = R.offsets(lengths)
    conv, ssm = conv.cpu().double().clone(), ssm.cpu().double().clone()
    for s, (a, b) in enumerate(zip(cu, cu[1:])):
        if a == b:
            continue
        old = (conv[s], ssm[s]) if starts[s] else (torch.zeros_like(conv[s]), torch.zeros_like(ssm[s]))
        mixed, _, conv[s] = R.conv(h[a:b, inner:inner + channels], c(m.weight), c(m.bias), old[0])
        x, bb, cc = mixed.split((inner, GROUPS * N, GROUPS * N), 1)
        out, _, ssm[s], _ = R.scan(x.view(-1, HEADS, p), h[a:b, inner + channels:inner + channels + HEADS], c(m.a), bb.view(-1, GROUPS, N), cc.view(-1, GROUPS, N),
                                   c(m.d), c(m.dt_bias), old[1])
        y[a:b] = R.gated_norm(out.flatten(1), h[a:b, :inner], c(m.norm_weight), m.norm_groups, m.eps)[0]
    return y, conv, ssm


def near(got, want):
    """three operators hand values over that are rounded to fp16 (2^-11 each, and as much within the scan), and the norm keeps their relative size"""
    got, want = got.cpu().double(), want
    assert (got - want).norm() <= 4 * 2.0 ** -11 * want.norm(), float((got - want).norm() / want.norm())


def test_a_serving_loop(gpu):
    """prompts, pieces of prompts and single tokens in one batch, requests that begin, pause and end"""
    from uniql_amd.state_space import StateSpaceStates
    m = mixer(gpu)
    states = StateSpaceStates.like(m, 4)
    states.conv.fill_(float("nan")), states.ssm.fill_(float("nan"))
    conv, ssm = states.conv.clone(), states.ssm.clone()
    had = [0, 0, 0, 0]
    for step, lengths in enumerate([[70, 3, 0, 1], [1, 1, 130, 1], [1, 0, 1, 65], [1, 1, 1, 1]]):
        h = projected(sum(lengths), gpu, seed=step)
        got = m(h, states, cu=ints(R.offsets(lengths), gpu), starts=ints(had, gpu))
        want, conv, ssm = in_64_bits(m, h, lengths, conv, ssm, had)
        near(got, want)
        near(states.ssm[[s for s in range(4) if had[s] or lengths[s]]], ssm[[s for s in range(4) if had[s] or lengths[s]]])
        had = [a + b for a, b in zip(had, lengths)]
        if step == 1:   # the last one ends, and another takes its place
            had[3] = 0
    # single tokens without offsets: the same states
    h = projected(4, gpu, seed=9)
    other = StateSpaceStates.like(m, 4)
    other.conv.copy_(states.conv), other.ssm.copy_(states.ssm)
    a = m(h, states)
    b = m(h, other, cu=ints([0, 1, 2, 3, 4], gpu))
    want, conv, ssm = in_64_bits(m, h, [1] * 4, conv, ssm, had)
    near(a, want), near(b, want)
    assert torch.equal(states.conv, other.conv)


def test_between_the_projections(gpu):
    """the 4-bit projections around it: a prompt at once, and as pieces"""
    from uniql_amd.quantize.quant_linear_layers import W4A16B16O16Linear
    from uniql_amd.state_space import StateSpaceStates
    torch.manual_seed(0)
    into = W4A16B16O16Linear.from_fp16(torch.nn.Linear(256, 512 + 2 * GROUPS * N + HEADS, bias=False).half().to(gpu)).to(gpu)
    out = W4A16B16O16Linear.from_fp16(torch.nn.Linear(256, 256, bias=False).half().to(gpu)).to(gpu)
    m = mixer(gpu, p=64)
    x = torch.randn(150, 256, device=gpu).half()
    h = into(x)
    whole = StateSpaceStates.like(m, 1)
    y = out(m(h, whole, cu=ints([0, 150], gpu), starts=ints([0], gpu)), residual=x)
    pieces, parts, at = StateSpaceStates.like(m, 1), [], 0
    for n in (1, 64, 2, 83):
        parts.append(m(h[at:at + n], pieces, cu=ints([0, n], gpu), starts=ints([at], gpu)))
        at += n
    z = out(torch.cat(parts), residual=x)
    want = in_64_bits(m, h, [150], whole.conv, whole.ssm, [0])[0]
    near(torch.cat(parts), want)
    near(y - x, (z - x).cpu().double())
    assert torch.equal(whole.conv, pieces.conv)
    within(pieces.ssm, whole.ssm.cpu().double(), 2.0 ** -18 * whole.ssm.abs().max().cpu().double().expand(whole.ssm.shape))


def test_next_to_a_cache(gpu):
    """offsets and starts from the pages; a request that they refuse keeps its states and is asked for again, one that ends makes room"""
    from uniql_amd.quantize.quant_kv_cache import KVPages
    from uniql_amd.state_space import StateSpaceStates
    m = mixer(gpu)
    states, pages = StateSpaceStates.like(m, 3), KVPages(8, 16, 3, 8, device=gpu)
    conv, ssm = states.conv.clone(), states.ssm.clone()
    for step, (new, refused) in enumerate((([40, 17, 0], [0, 0, 0]), ([1, 64, 2], [0, 1, 1]), ([-1, 60, 20], [0, 0, 0]), ([1, 1, 1], [0, 0, 0]))):
        starts = pages.lengths.clone()
        s = pages.assign(ints(new, gpu), 128)
        assert s.refused.tolist() == refused
        places = torch.where(s.refused > 0, -1, torch.arange(3, dtype=torch.int32, device=gpu))
        h = projected(128, gpu, seed=20 + step)
        got = m(h, states, cu=s.cu, places=places, starts=starts)
        cu, had = s.cu.tolist(), starts.tolist()
        for r in range(3):
            if refused[r] or new[r] <= 0:
                continue
            want, c, S = in_64_bits(m, h[cu[r]:cu[r + 1]], [new[r]], conv[r:r + 1], ssm[r:r + 1], [had[r]])
            near(got[cu[r]:cu[r + 1]], want)
            conv, ssm = conv.cpu().double(), ssm.cpu().double()
            conv[r], ssm[r] = c[0], S[0]
        near(states.ssm, ssm.cpu().double())


def test_without_states(gpu):
    m = mixer(gpu)
    h = projected(90, gpu)
    near(m(h, cu=ints([0, 40, 40, 90], gpu)), in_64_bits(m, h, [40, 0, 50], torch.zeros(3, 3, CHANNELS), torch.zeros(3, HEADS, P, N), [0] * 3)[0])
    with pytest.raises(RuntimeError, match="state"):
        m(h)


@pytest.mark.parametrize("p,n", [(8, 16), (12, 33), (100, 96), (64, 128), (54, 256), (1, 1)])
@pytest.mark.parametrize("in_place", [True, False])
def test_single_tokens_among_prompts(gpu, p, n, in_place):
    """each length next to each other, left out, beginning and continued; fewer sequences than four; offsets in front and rows behind"""
    for lengths in ([1, 5, 1, 0, 1, 130, 1, 64, 1], [1, 1, 1, 1, 1, 1], [1, 2, 1], [3, 0, 2, 65], [1], [0, 0, 0, 1]):
        pr = Problem(lengths, 4, 2, p, n, seed=11, first=2, behind=3)
        if len(lengths) > 4:
            pr.places[2] = -1
            pr.places[5] = -1
        check_scan(pr, gpu, in_place=in_place)


def test_more_heads_and_sequences_than_steps_take(gpu):
    check_scan(Problem([1] * 36 + [3, 1], 1 << 15, 1, 1, 1, seed=12), gpu)


@pytest.mark.parametrize("single", [True, False])
def test_graphs(gpu, single):
    """two graphs of the same layer, replayed in turn with eager work between; lengths and values change from replay to replay"""
    from uniql_amd.state_space import StateSpaceStates
    m = mixer(gpu)
    most, requests = (4, 4) if single else (700, 3)
    inputs = [projected(most, gpu, seed=s) for s in range(2)]
    cus = [ints([0, 1, 2, 3, 4] if single else [0, 300, 301, 700], gpu) for _ in range(2)]
    starts = ints([1] * requests, gpu)
    states = [StateSpaceStates.like(m, requests) for _ in range(2)]
    call = lambda h, s, cu: m(h, s, cu=None if single else cu, starts=starts)
    for s in states:
        call(inputs[0], s, cus[0])
        s.conv.zero_(), s.ssm.zero_()
    graphs, outs = [], []
    for h, s, cu in zip(inputs, states, cus):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(h, s, cu))
        graphs.append(g)
    mirror = [StateSpaceStates.like(m, requests) for _ in range(2)]
    for i, lengths in enumerate([[300, 1, 399], [0, 0, 700], [64, 65, 500], [1, 1, 1]]):
        for j in (0, 1):
            inputs[j].copy_(projected(most, gpu, seed=100 + 10 * i + j))
            if not single:
                cus[j].copy_(ints(R.offsets(lengths), gpu))
            graphs[j].replay()
        for j in (0, 1):
            want = call(inputs[j], mirror[j], cus[j])   # eager, on the same stream
            rows = most if single else sum(lengths)
            assert torch.equal(outs[j][:rows], want[:rows])
            assert torch.equal(states[j].ssm, mirror[j].ssm) and torch.equal(states[j].conv, mirror[j].conv)


def test_two_streams_at_once(gpu):
    pr = [Problem([900, 300], 2, 1, 12, 24, seed=s, decay=0.3) for s in (1, 2)]
    alone = [run_scan(p, gpu) for p in pr]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(gpu) for _ in pr], [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = run_scan(pr[i], gpu)
        torch.cuda.synchronize()
        for (y, st), (want_y, want_st) in zip(got, alone):
            assert torch.equal(st, want_st)
            assert torch.equal(y[:1200], want_y[:1200])


def test_rows_far_apart(gpu):
    """offsets beyond 2^31 elements: rows that still go straight to LDS, and rows too far apart for that"""
    from uniql_amd import ops
    for stride, rows in ((1 << 21, 1100), ((1 << 23) + 2, 270)):
        pr = Problem([rows], 1, 1, 8, 16, seed=3, starts=[0])
        buf = torch.empty(stride * rows, dtype=torch.float16, device=gpu)
        far = buf.as_strided((rows, pr.channels + 1), (stride, 1))
        far.copy_(torch.cat([pr.mixed, pr.dt], 1).to(gpu))
        x, b, c = far[:, :8].unflatten(1, (1, 8)), far[:, 8:24].unflatten(1, (1, 16)), far[:, 24:40].unflatten(1, (1, 16))
        y, tol, S, S_tol = pr.want_scan()
        state = pr.state.to(gpu)
        got = ops.state_space_scan(x, far[:, 40:41], pr.a.to(gpu), b, c, d=pr.d.to(gpu), dt_bias=pr.dt_bias.to(gpu), state=state, cu=ints(pr.cu, gpu),
                                   places=ints(pr.places, gpu), starts=ints([0], gpu))
        within(got, y, tol)
        within(state, S, S_tol)
        want, tol, _ = pr.want_conv()
        within(ops.causal_conv(far[:, :40], pr.weight.to(gpu), pr.bias.to(gpu), cu=ints(pr.cu, gpu)), want, tol)
        del buf, far, x, b, c


def test_rows_that_overlap(gpu):
    """x as windows of one sequence of numbers, whose last one is an infinity: it belongs to the last row alone"""
    from uniql_amd import ops
    for rows in (5, 70):
        pr = Problem([rows], 1, 1, 24, 16, seed=6, starts=[0])
        numbers = torch.randn(8 * (rows - 1) + 24, generator=torch.Generator().manual_seed(6)).half()
        windows = lambda t: t.as_strided((rows, 1, 24), (8, 24, 1))
        finite = numbers.clone()
        finite[-1] = 1
        numbers[-1] = float("inf")
        on = lambda t: on_gpu(t, gpu)
        got = []
        for t in (finite, numbers):
            state = torch.zeros(1, 1, 24, 16, device=gpu)
            got.append((ops.state_space_scan(windows(t.to(gpu)), on(pr.dt), pr.a.to(gpu), on(pr.b), on(pr.c), dt_bias=pr.dt_bias.to(gpu), state=state,
                                             cu=ints([0, rows], gpu)), state))
        want, tol, S, S_tol = R.scan(windows(finite).contiguous(), pr.dt, pr.a, pr.b, pr.c, None, pr.dt_bias, torch.zeros(1, 24, 16))
        within(got[0][0], want, tol), within(got[0][1][0], S, S_tol)
        # all but the last channel of the last row, and of the state
        within(got[1][0][:-1], want[:-1], tol[:-1]), within(got[1][0][-1, :, :-1], want[-1, :, :-1], tol[-1, :, :-1])
        within(got[1][1][0, :, :-1], S[:, :-1], S_tol[:, :-1])
        assert not got[1][1][0, 0, -1].isfinite().any() and not got[1][0][-1, 0, -1].isfinite()


def test_places_far_apart(gpu):
    """a pool of more than 2^31 numbers"""
    from uniql_amd import ops
    heads, p, n, places = 16, 64, 128, 16500
    state = torch.zeros(places, heads, p, n, device=gpu)
    for cu in (None, [0, 1, 66]):
        rows = 2 if cu is None else 66
        pr = Problem([1, 1] if cu is None else [1, 65], heads, 1, p, n, seed=4, starts=[1, 1], spare=0)
        pr.places = [0, 1]
        at = [16450, 3]
        state[at[0]], state[at[1]] = pr.state[0].to(gpu), pr.state[1].to(gpu)
        y, tol, S, S_tol = pr.want_scan()
        got = ops.state_space_scan(on_gpu(pr.x, gpu), on_gpu(pr.dt, gpu), pr.a.to(gpu), on_gpu(pr.b, gpu), on_gpu(pr.c, gpu), d=pr.d.to(gpu),
                                   dt_bias=pr.dt_bias.to(gpu), state=state, cu=ints(cu, gpu), places=ints(at, gpu))
        assert got.shape[0] == rows
        within(got, y, tol)
        within(state[at], S, S_tol)
    assert not state[16451:].any() and not state[4:16450].any()


def refuses(match, f, *args, **kw):
    with pytest.raises(RuntimeError, match=match):
        f(*args, **kw)


def test_conv_refusals(gpu):
    from uniql_amd import ops
    x, w = torch.zeros(6, 16, dtype=torch.float16, device=gpu), torch.zeros(16, 4, dtype=torch.float16, device=gpu)
    state, cu = torch.zeros(3, 3, 16, dtype=torch.float16, device=gpu), ints([0, 2, 6], gpu)
    f = ops.causal_conv
    ok = dict(state=state, cu=cu)
    f(x, w, **ok)
    refuses("GPU", f, x.cpu(), w, **ok)
    refuses("float16", f, x.float(), w, **ok)
    refuses("unit stride", f, torch.zeros(16, 6, dtype=torch.float16, device=gpu).t(), w, **ok)
    refuses("2 to 4", f, x, torch.zeros(16, 5, dtype=torch.float16, device=gpu), **ok)
    refuses("2 to 4", f, x, w[:8], **ok)
    refuses("bias", f, x, w, w[:8, 0].contiguous(), **ok)
    refuses("needs a state", f, x, w)
    refuses("state must be", f, x, w, state=state[:, :2].contiguous(), cu=cu)
    refuses("contiguous Float|contiguous Half", f, x, w, state=state.float(), cu=cu)
    refuses("starts without", f, x, w, cu=cu, starts=ints([0, 0], gpu))
    refuses("starts must", f, x, w, starts=ints([0], gpu), **ok)
    refuses("places must", f, x, w, places=ints([0, 1, 2], gpu), **ok)
    refuses("one place per sequence", f, x, w, state=state[:1], cu=cu)
    refuses("one place per sequence", f, x, w, state=state)
    refuses("same places", f, x, w, state_out=state[:2].clone(), **ok)
    refuses("share no memory", f, x, w, state=state[:2], state_out=state[1:], cu=ints([0, 6], gpu))
    refuses("out must not be x", f, x, w, out=x, **ok)
    refuses("out must be", f, x, w, out=x[:5], **ok)
    refuses("cu must", f, x, w, state=state, cu=ints([], gpu))
    assert f(x[:0], w, state=state, cu=ints([0, 0], gpu)).shape == (0, 16)


def test_scan_refusals(gpu):
    from uniql_amd import ops
    h = lambda *s: torch.zeros(*s, dtype=torch.float16, device=gpu)
    x, dt, b, c, a = h(6, 4, 8), h(6, 4), h(6, 2, 16), h(6, 2, 16), torch.zeros(4, device=gpu)
    state, cu = torch.zeros(3, 4, 8, 16, device=gpu), ints([0, 2, 6], gpu)
    f = ops.state_space_scan
    ok = dict(state=state, cu=cu)
    f(x, dt, a, b, c, **ok)
    refuses("GPU", f, x.cpu(), dt, a, b, c, **ok)
    refuses("float16", f, x.float(), dt, a, b, c, **ok)
    refuses("dt must", f, x, dt[:5], a, b, c, **ok)
    refuses("dt must", f, x, dt.float(), a, b, c, **ok)
    refuses("a must", f, x, dt, a.half(), b, c, **ok)
    refuses("per head", f, x, dt, a[:3].contiguous(), b, c, **ok)
    refuses("same groups", f, x, dt, a, b, c[:, :1], **ok)
    refuses("multiple", f, x, dt, a, h(6, 3, 16), h(6, 3, 16), **ok)
    refuses("1 to 128", f, h(6, 4, 129), dt, a, b, c, cu=cu)
    refuses("1 to 256", f, x, dt, a, h(6, 2, 257), h(6, 2, 257), cu=cu)
    refuses("dt_limit", f, x, dt, a, b, c, dt_limit=(-0.1, 1.0), **ok)
    refuses("dt_limit", f, x, dt, a, b, c, dt_limit=(1.0, 0.5), **ok)
    refuses("state must be", f, x, dt, a, b, c, state=state[:, :2].contiguous(), cu=cu)
    refuses("needs a state", f, x, dt, a, b, c)
    refuses("d must", f, x, dt, a, b, c, d=a.half(), **ok)
    refuses("out must not", f, x, dt, a, b, c, out=x, **ok)
    refuses("out must be", f, x, dt, a, b, c, out=h(6, 4, 9), **ok)
    refuses("share no memory", f, x, dt, a, b, c, state=state[:2], state_out=state[1:], cu=ints([0, 6], gpu))
    assert f(x[:0], dt[:0], a, b[:0], c[:0], state=state, cu=ints([0, 0], gpu)).shape == (0, 4, 8)


def test_outputs_in_the_inputs(gpu):
    from uniql_amd import ops
    memory = torch.zeros(4096, dtype=torch.int32, device=gpu)
    halves, floats = memory.view(torch.float16), memory.view(torch.float32)
    small = memory[:3].copy_(ints([0, 2, 6], gpu))
    h = lambda *s: torch.zeros(*s, dtype=torch.float16, device=gpu)
    x, w, b = h(6, 16), h(16, 4), h(6, 1, 8)
    for kw in (dict(cu=small), dict(cu=ints([0, 2, 6], gpu), places=small[:2]), dict(cu=ints([0, 2, 6], gpu), starts=small[:2])):
        refuses("share memory", ops.causal_conv, x, w, state=halves[:96].view(2, 3, 16), **kw)
        refuses("share memory", ops.causal_conv, x, w, state=h(2, 3, 16), out=halves[:96].view(6, 16), **kw)
        refuses("share memory", ops.state_space_scan, x.view(6, 2, 8), h(6, 2), torch.zeros(2, device=gpu), b, b, state=floats[:256].view(2, 2, 8, 8), **kw)
        refuses("share memory", ops.state_space_scan, x.view(6, 2, 8), h(6, 2), torch.zeros(2, device=gpu), b, b, state=torch.zeros(2, 2, 8, 8, device=gpu),
                out=halves[:96].view(6, 2, 8), **kw)
    refuses("share memory", ops.causal_conv, x, halves[:64].view(16, 4), cu=ints([0, 6], gpu), out=halves[:96].view(6, 16))
    refuses("share memory", ops.state_space_scan, x.view(6, 2, 8), h(6, 2), floats[:2], b, b, state=floats[:128].view(1, 2, 8, 8), cu=ints([0, 6], gpu))


def test_norm_refusals(gpu):
    from uniql_amd import ops
    x = torch.zeros(6, 16, dtype=torch.float16, device=gpu)
    w, f = x[0].contiguous(), ops.gated_group_norm
    f(x, x, w, 2)
    refuses("GPU", f, x.cpu(), x, w)
    refuses("x's shape", f, x, x[:5], w)
    refuses("weight", f, x, x, w[:8].contiguous())
    refuses("divide", f, x, x, w, 3)
    refuses("divide", f, x, x, w, 0)
    refuses("negative", f, x, x, w, 2, -1.0)
    refuses("itself", f, x, x, w, 2, out=torch.zeros(7, 16, dtype=torch.float16, device=gpu)[1:].as_strided((6, 16), (8, 1)))
    big = torch.zeros(8, 16, dtype=torch.float16, device=gpu)
    refuses("share no memory", f, big[:6], x, w, 2, out=big[1:7])
    assert f(x[:0], x[:0], w).shape == (0, 16)
