"""Attention over packed prompts against 64-bit arithmetic."""
import pytest
import torch

from tests.attention_reference import attention, bound

pytestmark = pytest.mark.gpu


def offsets(lengths, first=0):
    out = [first]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def problem(lens_q, lens_k, h, g, d, e, seed=0, sharp=1.0, first=0, behind=0, shift=0):
    """q, k, v: ranges of one buffer each row of which is `shift` elements longer than it has to be"""
    gen = torch.Generator().manual_seed(seed)
    cu_q, cu_k = offsets(lens_q, first), offsets(lens_k, first)
    rows_q, rows_k = cu_q[-1] + behind, cu_k[-1] + behind
    buf = torch.randn(rows_q * (h * d + shift) + shift, generator=gen).mul_(sharp).half()
    kv = torch.randn(rows_k * (g * (d + e) + shift) + shift, generator=gen).half()
    q = buf[shift:].view(rows_q, -1)[:, :h * d].view(rows_q, h, d)
    rows = kv[shift:].view(rows_k, -1)
    return q, rows[:, :g * d].view(rows_k, g, d), rows[:, g * d:g * (d + e)].view(rows_k, g, e), cu_q, cu_k


def on_gpu(t, dev):
    """a copy on the device that lies as t does"""
    base = t._base if t._base is not None else t
    return base.to(dev).as_strided(t.size(), t.stride(), t.storage_offset())


def reference(q, k, v, cu_q, cu_k, scale, causal=True):
    o = torch.zeros(q.shape[0], q.shape[1], v.shape[2], dtype=torch.float64)
    tol = torch.zeros_like(o)
    for a, b, c, d in zip(cu_q, cu_q[1:], cu_k, cu_k[1:]):
        first = d - c - (b - a) + 1 if causal else d - c
        part = attention(q[a:b], k[c:d], v[c:d], scale, first) if causal else \
            tuple(torch.cat(x) for x in zip(*[attention(q[i:i + 1], k[c:d], v[c:d], scale, first) for i in range(a, b)])) if b > a else None
        if part is None:
            continue
        o[a:b], tol[a:b] = part[0], bound(*part, d - c)
    return o, tol


def run(dev, q, k, v, cu_q, cu_k, **kw):
    from uniql_amd.attention import prompt_attention
    t = lambda c: torch.tensor(c, dtype=torch.int32, device=dev)
    return prompt_attention(on_gpu(q, dev), on_gpu(k, dev), on_gpu(v, dev), t(cu_q), None if cu_k is None else t(cu_k), **kw)


CASES = [
    ([1], 1, 1, 1, 1), ([1, 2, 0, 3], 2, 1, 8, 8), ([63, 64, 65], 4, 2, 64, 64), ([127, 1, 129], 2, 2, 128, 128), ([300], 4, 1, 108, 100),
    ([31, 33, 0, 0, 97], 6, 3, 126, 34), ([257], 2, 1, 96, 128), ([40, 513], 3, 1, 32, 96), ([200], 5, 5, 33, 17), ([260, 5], 8, 1, 128, 64),
]


@pytest.mark.parametrize("lengths,h,g,d,e", CASES)
@pytest.mark.parametrize("shift", [0, 1, 8])
def test_prompts(gpu, lengths, h, g, d, e, shift):
    q, k, v, cu, _ = problem(lengths, lengths, h, g, d, e, seed=len(lengths) + d, sharp=1.5, shift=shift)
    want, tol = reference(q, k, v, cu, cu, d ** -0.5)
    got = run(gpu, q, k, v, cu, None).cpu().double()
    assert got.shape == want.shape
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() - tol).max())


@pytest.mark.parametrize("lens_q,lens_k,h,g,d,e", [
    ([5, 1, 20, 3, 0, 4], [40, 0, 10, 3, 9, 130], 4, 2, 64, 64), ([70, 1], [300, 257], 2, 1, 128, 128), ([130], [64], 2, 2, 100, 36),
    ([1, 1, 1], [1, 100, 515], 8, 2, 128, 128),
])
@pytest.mark.parametrize("causal", [True, False])
def test_keys_of_other_lengths_than_queries(gpu, lens_q, lens_k, h, g, d, e, causal):
    """a prompt taken in pieces; rows that see no key at all are zeros"""
    q, k, v, cu_q, cu_k = problem(lens_q, lens_k, h, g, d, e, seed=d)
    want, tol = reference(q, k, v, cu_q, cu_k, 0.11, causal)
    got = run(gpu, q, k, v, cu_q, cu_k, causal=causal, scale=0.11).cpu().double()
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() - tol).max())
    if causal and lens_q[0] == 130:
        assert (got[:66] == 0).all()


@pytest.mark.parametrize("sharp,scale", [(40.0, 1.0), (1e-3, 1e-3), (2.0, 0.0), (3.0, -0.3)])
def test_sharp_flat_and_negative_scores(gpu, sharp, scale):
    q, k, v, cu, _ = problem([150, 30], [150, 30], 2, 1, 64, 48, seed=3, sharp=sharp)
    want, tol = reference(q, k, v, cu, cu, scale)
    if scale < 0:
        tol = reference(q, k, v, cu, cu, -scale)[1] + (tol - tol) + 2 ** -10 * want.abs().amax()
    got = run(gpu, q, k, v, cu, None, scale=scale).cpu().double()
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() - tol).max())


def test_scores_that_grow_along_the_keys(gpu):
    """the running maximum rises with every key, and falls: every weight is rescaled many times"""
    for rising in (True, False):
        n = 400
        q = torch.ones(n, 2, 16).half()
        ramp = torch.arange(n, dtype=torch.float32) * (1 if rising else -1) / 16
        k = (ramp.view(n, 1, 1) * torch.ones(n, 1, 16)).half()
        v = torch.randn(n, 1, 32, generator=torch.Generator().manual_seed(1)).half()
        want, tol = reference(q, k, v, [0, n], [0, n], 0.5)
        got = run(gpu, q, k, v, [0, n], None, scale=0.5).cpu().double()
        assert ((got - want).abs() <= tol).all()


def test_rows_outside_the_sequences_are_left_alone(gpu):
    q, k, v, cu, _ = problem([50, 0, 90], [50, 0, 90], 2, 2, 64, 40, first=3, behind=70)
    out = torch.full((213, 2, 48), 5.0, device=gpu).half()[:, :, :40]
    want, tol = reference(q, k, v, cu, cu, 0.125)
    got = run(gpu, q, k, v, cu, None, scale=0.125, out=out)
    assert got.data_ptr() == out.data_ptr()
    got = got.cpu().double()
    assert (got[:3] == 5).all() and (got[143:] == 5).all()
    assert ((got - want).abs() <= tol)[3:143].all()
    assert (out._base[:, :, 40:] == 5).all()


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan"), 65504.0])
@pytest.mark.parametrize("d,e", [(64, 64), (108, 100)])
def test_what_a_row_does_not_see_does_not_matter(gpu, bad, d, e):
    """later keys, other sequences and rows behind them hold infinities and NaN"""
    q, k, v, cu, _ = problem([40, 75, 20], [40, 75, 20], 4, 2, d, e, seed=9, first=2, behind=30)
    want, tol = reference(q, k, v, cu, cu, 0.1)
    kb, vb = k.clone(), v.clone()
    for t in (kb, vb):
        t[:2], t[137:] = bad, bad                 # outside every sequence
        t[2:42] = bad                             # the first sequence
        t[42 + 60:42 + 75] = bad                  # the last keys of the second
    qb = q.clone()
    qb[2:42] = bad
    got = run(gpu, qb, kb, vb, cu, None, scale=0.1, out=torch.zeros(q.shape[0], 4, e, device=gpu).half()).cpu().double()
    for rows in (slice(42, 102), slice(117, 137)):
        assert ((got[rows] - want[rows]).abs() <= tol[rows]).all()


def test_infinities_and_nan_that_a_row_sees(gpu):
    """as 64-bit arithmetic has it: an infinite value or a NaN among the keys or values shows in every row that sees it"""
    q, k, v, cu, _ = problem([90], [90], 2, 1, 64, 64, seed=2)
    k = k.clone()
    v = v.clone()
    v[50, 0, 7] = float("nan")
    v[60, 0, 9] = float("inf")
    k[70, 0, 3] = float("nan")
    got = run(gpu, q, k, v, [0, 90], None).cpu()
    assert got[:50].isfinite().all() and got[50:, :, 7].isnan().all() and got[50:60, :, 8:].isfinite().all()
    assert not got[60:, :, 9].isfinite().any() and got[60:70, :, 10:].isfinite().all() and got[70:].isnan().all()


def test_offsets_that_do_not_describe_the_rows(gpu):
    """offsets below 0, beyond the rows or falling: nothing outside the tensors is read or written"""
    q, k, v, _, _ = problem([64], [64], 2, 1, 64, 64)
    for cu in ([-5, 30, 200], [10, 5, 64], [0, 2 ** 31 - 1, 2 ** 31 - 1], [-2 ** 31, -1, 64], [64, 64, 64]):
        run(gpu, q, k, v, cu, cu)
        run(gpu, q, k, v, [0, 32, 64], cu)
        run(gpu, q, k, v, cu, [0, 32, 64], causal=False)
    torch.cuda.synchronize()


def test_strides_beyond_32_bits(gpu):
    """rows so far apart that their offsets pass 2^31 elements"""
    q, k, v, cu, _ = problem([70], [70], 2, 1, 64, 64, seed=4)
    want, tol = reference(q, k, v, cu, cu, 0.125)
    far = 1 << 25
    big = torch.empty(70 * far, dtype=torch.float16, device=gpu)
    views = []
    for at, t in ((0, q), (1000, k), (2000, v)):
        w = big.as_strided(t.shape, (far, t.shape[2], 1), at)
        w.copy_(t.to(gpu))
        views.append(w)
    out = big.as_strided((70, 2, 64), (far, 64, 1), 4000)
    from uniql_amd.attention import prompt_attention
    prompt_attention(*views, torch.tensor(cu, dtype=torch.int32, device=gpu), scale=0.125, out=out)
    assert ((out.cpu().double() - want).abs() <= tol).all()


def test_same_result_every_time_and_on_another_stream_and_captured(gpu):
    from uniql_amd.attention import prompt_attention
    q, k, v, cu, _ = problem([500, 3, 77], [500, 3, 77], 4, 2, 128, 128)
    q, k, v = (t.to(gpu) for t in (q, k, v))
    cu = torch.tensor(cu, dtype=torch.int32, device=gpu)
    first = prompt_attention(q, k, v, cu)
    assert torch.equal(first, prompt_attention(q, k, v, cu))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = prompt_attention(q, k, v, cu)
    stream.synchronize()
    assert torch.equal(first, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = prompt_attention(q, k, v, cu)
    for i in range(4):
        q.copy_(torch.randn_like(q))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, prompt_attention(q, k, v, cu))


def test_refusals(gpu):
    from uniql_amd.attention import prompt_attention
    x = torch.zeros(8, 4, 64, dtype=torch.float16, device=gpu)
    cu = torch.tensor([0, 8], dtype=torch.int32, device=gpu)
    for args, kw, words in [
        ((x.float(), x, x, cu), {}, "float16"), ((x.cpu(), x, x, cu), {}, "GPU"), ((x, x.cpu(), x, cu), {}, "GPU"),
        ((x[:, :3], x[:, :2], x[:, :2], cu), {}, "multiple"), ((x, x[:, :, :32], x, cu), {}, "one width"),
        ((x, x, x[:4], cu), {}, "same rows"), ((x, x, x, cu.long()), {}, "cu_q"), ((x, x, x, cu[:0]), {}, "cu_q"),
        ((x, x, x, cu, cu[:1]), {}, "same number"), ((x.transpose(1, 2), x, x, cu), {}, "unit stride"),
        ((x, x, x, cu), dict(out=x[:, :, :32]), "out must be"), ((x, x, x, cu), dict(out=x[:1].expand(8, 4, 64)), "overlaps"),
        ((torch.zeros(8, 2, 130, dtype=torch.float16, device=gpu),) * 3 + (cu,), {}, "128 wide"),
    ]:
        with pytest.raises(RuntimeError, match=words):
            prompt_attention(*args, **kw)
    assert prompt_attention(x[:0], x, x, cu).shape == (0, 4, 64)


@pytest.mark.parametrize("count", [63, 64, 65, 200])
def test_many_sequences(gpu, count):
    """more sequences than a wave has lanes, most of them shorter than a tile of rows"""
    lengths = torch.randint(0, 40, (count,), generator=torch.Generator().manual_seed(count)).tolist()
    lengths[count // 3] = 300
    q, k, v, cu, _ = problem(lengths, lengths, 6, 2, 32, 40, seed=count, first=1, behind=3)
    want, tol = reference(q, k, v, cu, cu, 0.2)
    got = run(gpu, q, k, v, cu, None, scale=0.2).cpu().double()
    assert ((got - want).abs() <= tol)[1:-3].all()


@pytest.mark.parametrize("h,g", [(7, 7), (12, 4), (20, 4), (33, 1), (64, 1), (130, 1)])
def test_groups_of_every_kind(gpu, h, g):
    q, k, v, cu, _ = problem([70, 3, 140], [70, 3, 140], h, g, 48, 32, seed=h)
    want, tol = reference(q, k, v, cu, cu, 0.15)
    got = run(gpu, q, k, v, cu, None, scale=0.15).cpu().double()
    assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("d,e", [(2, 2), (10, 12), (30, 62), (66, 34), (94, 96), (98, 126), (126, 130 - 2), (64, 66)])
@pytest.mark.parametrize("neighbour", [float("nan"), float("inf")])
def test_rows_whose_neighbours_are_no_numbers(gpu, d, e, neighbour):
    """even widths, pieces of which reach into other columns of the same rows: what those hold does not matter"""
    n = 150
    gen = torch.Generator().manual_seed(d + e)
    row = 2 * d + 2 * e + 8
    buf = torch.full((n, row), neighbour).half()
    q = torch.randn(n, 2, d, generator=gen).half()
    k, v = buf[:, 2:2 + d].view(n, 1, d), buf[:, d + 4:d + 4 + e].view(n, 1, e)
    k.copy_(torch.randn(n, 1, d, generator=gen))
    v.copy_(torch.randn(n, 1, e, generator=gen))
    want, tol = reference(q, k, v, [0, n], [0, n], 0.2)
    got = run(gpu, q, k, v, [0, n], None, scale=0.2).cpu().double()
    assert ((got - want).abs() <= tol).all()


def test_a_scale_that_is_no_number_and_an_output_that_is_an_input(gpu):
    from uniql_amd.attention import prompt_attention
    x = torch.zeros(8, 4, 64, dtype=torch.float16, device=gpu)
    cu = torch.tensor([0, 8], dtype=torch.int32, device=gpu)
    for scale in (float("nan"), float("-inf"), 1e300):
        with pytest.raises(RuntimeError):
            prompt_attention(x, x, x, cu, scale=scale)
    with pytest.raises(RuntimeError, match="must not be"):
        prompt_attention(x, x, x, cu, out=x)
    with pytest.raises(RuntimeError, match="must not be"):
        prompt_attention(x.clone(), x, x.clone(), cu, out=x)


def test_many_small_weights_beside_a_large_one(gpu):
    """one key has the weight 1 and the value -1, 60000 have 2^-25.1 and 1: together 0.0017, each below what is left of an fp16 number
    scaled to 1.  Rounding: of the large weight 2^-11, of the small ones' sum (2^-25 of 2^-19.1) 3e-5, of the result 2^-12."""
    from uniql_amd.attention import prompt_attention
    n = 60001
    k = torch.zeros(n, 1, 64).half()
    k[100] = 1.0
    v = torch.ones(n, 1, 64).half()
    v[100] = -1.0
    cu = [torch.tensor([0, x], dtype=torch.int32, device=gpu) for x in (1, n)]
    got = prompt_attention(torch.ones(1, 2, 64, device=gpu).half(), k.to(gpu), v.to(gpu), cu[0], cu[1], scale=25.1 * 0.6931471805599453 / 64)
    weight = 2.0 ** -25.1
    want = (-1 + (n - 1) * weight) / (1 + (n - 1) * weight)
    assert (got.cpu().double() - want).abs().max() <= 2 ** -10, float((got.cpu().double() - want).abs().max())
