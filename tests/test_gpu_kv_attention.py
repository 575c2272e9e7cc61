"""Attention over the paged 4-bit cache against 64-bit arithmetic on the values that it holds."""
import pytest
import torch

from tests.attention_reference import as_held, attention, bound

pytestmark = pytest.mark.gpu


class Problem:
    """lengths: tokens of each request in the cache; tokens: rows of q of each.  Pages lie in no order among twice as many, and what
    no request holds is full of codes and of scales that are infinite or NaN."""

    def __init__(self, dev, lengths, tokens, h, g, d, e, page, seed=0, sharp=1.5, k_of=None, v_of=None, extra_columns=1):
        from uniql_amd.quantize.quant_kv_cache import W4KVCache
        gen = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in lengths]
        columns = max(need) + extra_columns
        pages = 2 * sum(need) + 2
        order = torch.randperm(pages, generator=gen).to(torch.int32).tolist()
        self.table = torch.full((len(lengths), columns), -1, dtype=torch.int32)
        for r, n in enumerate(need):
            for j in range(n):
                self.table[r, j] = order.pop()
        self.cache = W4KVCache(pages, page, g, d, e, device=dev)
        for t in (self.cache.k_codes, self.cache.v_codes):
            t.copy_(torch.randint(-2 ** 31, 2 ** 31 - 1, t.shape, generator=gen).int())
        self.cache.k_scales.fill_(float("nan"))
        self.cache.v_scales.fill_(float("inf"))
        self.lengths, self.tokens = lengths, tokens
        self.k = [torch.randn(n, g, d, generator=gen).half() for n in lengths]
        self.v = [torch.randn(n, g, e, generator=gen).half() for n in lengths]
        for r in range(len(lengths)):
            if k_of:
                self.k[r] = k_of(self.k[r])
            if v_of:
                self.v[r] = v_of(self.v[r])
            pos = torch.arange(lengths[r])
            slots = self.table[r].long()[pos // page] * page + pos % page
            self.cache.store(self.k[r].to(dev), self.v[r].to(dev), slots.to(dev))
        cu = [0]
        for t in tokens:
            cu.append(cu[-1] + t)
        self.cu = cu
        self.q = (torch.randn(cu[-1], h, d, generator=gen) * sharp).half()
        self.dev, self.e = dev, e

    def on_gpu(self):
        t = lambda v: torch.tensor(v, dtype=torch.int32, device=self.dev)
        return self.q.to(self.dev), self.table.to(self.dev), t(self.lengths), None if set(self.tokens) == {1} else t(self.cu)

    def run(self, **kw):
        q, table, lengths, cu = self.on_gpu()
        return self.cache.attend(q, table, lengths, cu_q=cu, **kw)

    def check(self, got, scale):
        got = got.cpu().double()
        for r, n in enumerate(self.lengths):
            a, b = self.cu[r], self.cu[r + 1]
            if a == b:
                continue
            k, v = as_held(self.k[r])[0], as_held(self.v[r])
            first = n - (b - a) + 1
            o, mean_abs, spread = attention(self.q[a:b], k, v[0], scale, first)
            held = attention(self.q[a:b], k, v[1].unsqueeze(-1), scale, first)[0]
            tol = bound(o, mean_abs, spread, n, held)
            err = (got[a:b] - o).abs()
            assert (err <= tol).all(), (r, n, float((err - tol).max()), float(err.max()))


CASES = [
    ([1], [1], 1, 1, 1, 1, 16), ([1, 17, 16, 15], [1] * 4, 4, 2, 64, 64, 16), ([300, 33], [1, 1], 8, 2, 128, 128, 64),
    ([64, 65, 63, 128, 127, 129], [1] * 6, 8, 1, 128, 128, 32), ([1000], [1], 28, 4, 128, 128, 128), ([70, 5, 400], [1] * 3, 6, 6, 108, 100, 32),
    ([513, 2], [1, 1], 4, 1, 33, 126, 256), ([40, 100], [1, 1], 3, 3, 96, 31, 16), ([2000, 1, 500], [1] * 3, 32, 8, 128, 128, 16),
    ([7, 250], [1, 1], 20, 1, 64, 96, 16), ([90], [1], 40, 1, 70, 128, 16), ([4100], [1], 4, 1, 128, 128, 64),
    # several rows a request: causal at the end
    ([40, 300, 9], [5, 5, 5], 8, 2, 128, 128, 64), ([40, 20, 33, 700], [1, 20, 0, 37], 4, 4, 108, 100, 32), ([256], [100], 8, 2, 64, 64, 16),
    ([5, 3, 8], [7, 3, 1], 4, 2, 64, 64, 16),
]


@pytest.mark.parametrize("lengths,tokens,h,g,d,e,page", CASES)
def test_attention_over_the_cache(gpu, lengths, tokens, h, g, d, e, page):
    p = Problem(gpu, lengths, tokens, h, g, d, e, page, seed=d + h)
    p.check(p.run(), d ** -0.5)


def test_rows_that_see_nothing(gpu):
    """requests without tokens in the cache, and more rows than tokens (a request that was refused)"""
    p = Problem(gpu, [0, 3, 0, 20], [1, 5, 2, 1], 8, 2, 64, 40, 16)
    got = p.run()
    p.check(got, 0.125)
    assert (got[0] == 0).all() and (got[1:3] == 0).all() and (got[6:8] == 0).all()
    p = Problem(gpu, [0, 3], [1, 1], 8, 2, 64, 40, 16)
    got = p.run()
    p.check(got, 0.125)
    assert (got[0] == 0).all()


@pytest.mark.parametrize("size", [1e-6, 1e-3, 1.0, 4000.0])
def test_values_of_very_different_sizes(gpu, size):
    """value vectors from tiny to huge in one request, and all of one size near fp16's ends"""
    p = Problem(gpu, [333], [1], 4, 2, 64, 64, 16, v_of=lambda v: (v.float() * size).half())
    p.check(p.run(), 0.125)
    sizes = 10.0 ** torch.linspace(-4, 3, 333).view(-1, 1, 1)
    p = Problem(gpu, [333], [1], 4, 2, 64, 64, 16, v_of=lambda v: (v.float() * sizes * size / 4000).half())
    p.check(p.run(), 0.125)
    p = Problem(gpu, [333], [1], 4, 2, 64, 64, 16, v_of=lambda v: (v.float() * sizes.flip(0) * size / 4000).half())
    p.check(p.run(), 0.125)


@pytest.mark.parametrize("sharp,scale", [(30.0, 1.0), (1.0, 0.0), (1.0, -0.2)])
def test_sharp_flat_and_negative_scores(gpu, sharp, scale):
    p = Problem(gpu, [777, 130], [1, 1], 4, 1, 64, 64, 32, sharp=sharp)
    if scale < 0:   # the tolerance takes a positive scale: turn the queries instead
        got = p.run(scale=scale)
        p.q = -p.q
        p.check(got, -scale)
    else:
        p.check(p.run(scale=scale), scale)


def test_vectors_of_zeros(gpu):
    p = Problem(gpu, [100, 50], [1, 1], 4, 2, 64, 64, 16, k_of=torch.zeros_like, v_of=torch.zeros_like)
    got = p.run()
    assert (got == 0).all()
    p = Problem(gpu, [100, 50], [1, 1], 4, 2, 64, 64, 16, k_of=lambda k: torch.where(torch.arange(k.shape[0]).view(-1, 1, 1) % 3 > 0, k, 0 * k),
                v_of=lambda v: torch.where(torch.arange(v.shape[0]).view(-1, 1, 1) % 2 > 0, v, 0 * v))
    p.check(p.run(), 0.125)


def test_infinities_and_nan_show_where_they_are_seen(gpu):
    def spoil(at, what):
        def f(x):
            x = x.clone()
            x[at, 0, 1] = what
            return x
        return f
    for kw in (dict(k_of=spoil(60, float("inf"))), dict(k_of=spoil(60, float("nan"))), dict(v_of=spoil(60, float("-inf")))):
        p = Problem(gpu, [64, 80], [6, 1], 4, 2, 64, 64, 16, **kw)
        got = p.run().cpu()
        # request 0's rows see 59 .. 64 positions: the last two see position 60, heads 0 and 1 belong to the spoilt vector
        assert got[:2].isfinite().all() and got[2:6, :2].isnan().all() == got[2:6, :2].isnan().all()
        limits = [64 - 6 + i + 1 for i in range(6)]
        for i, seen in enumerate(limits):
            assert got[i, 2:].isfinite().all()
            assert got[i, :2].isnan().all() if seen > 60 else got[i, :2].isfinite().all()
        assert got[6, :2].isnan().all() and got[6, 2:].isfinite().all()


def test_page_numbers_outside_the_pool(gpu):
    """within a request's length they make the rows that see them NaN; behind it they do not matter"""
    for bad in (-1, 10 ** 9, -2 ** 31, 2 ** 31 - 1):
        p = Problem(gpu, [64, 100, 30], [2, 1, 1], 4, 2, 64, 64, 16, extra_columns=3)
        good = p.run()
        p.table[1, 3] = bad
        p.table[0, 4:] = bad
        p.table[2, 2:] = bad
        got = p.run()
        assert got[2].isnan().all() and torch.equal(got[:2], good[:2]) and torch.equal(got[3], good[3])
    p.table[:] = 5
    p.lengths = [2 ** 31 - 1, -4, 10 ** 6]   # beyond the table's room and below 0
    p.run()
    torch.cuda.synchronize()


def test_offsets_that_do_not_describe_the_rows(gpu):
    p = Problem(gpu, [64, 30], [3, 2], 4, 2, 64, 64, 16)
    q, table, lengths, _ = p.on_gpu()
    for cu in ([-5, 3, 2000], [4, 2, 5], [0, 2 ** 31 - 1, 2 ** 31 - 1], [-2 ** 31, 0, 5], [5, 5, 5]):
        p.cache.attend(q, table, lengths, cu_q=torch.tensor(cu, dtype=torch.int32, device=gpu))
    torch.cuda.synchronize()


def test_rows_outside_the_requests_and_strided_tensors(gpu):
    p = Problem(gpu, [64, 30], [3, 2], 4, 2, 72, 40, 16)
    want = p.run()
    q, table, lengths, _ = p.on_gpu()
    wide = torch.randn(12, 4 * 72 + 5, device=gpu).half()
    rows = wide[:, 3:3 + 4 * 72].unflatten(1, (4, 72))
    rows[4:9] = q
    out = torch.full((12, 4, 50), 3.0, device=gpu).half()
    got = p.cache.attend(rows, table, lengths, cu_q=torch.tensor([4, 7, 9], dtype=torch.int32, device=gpu), out=out[:, :, 1:41])
    assert got.data_ptr() == out[:, :, 1:].data_ptr()
    assert torch.equal(out[4:9, :, 1:41], want)
    out[4:9, :, 1:41] = 3.0
    assert (out == 3).all()


def test_places_beyond_32_bits(gpu):
    """a pool whose codes pass 2^31 words"""
    from uniql_amd.quantize.quant_kv_cache import W4KVCache
    small = Problem(gpu, [600, 300], [1, 1], 16, 8, 128, 128, 256)
    pages = 66000
    cache = W4KVCache(1, 256, 8, 128, 128, device=gpu)
    cache.k_codes = torch.empty(pages, 8, 256, 16, dtype=torch.int32, device=gpu)
    cache.v_codes = torch.empty(pages, 8, 64, 16, 4, dtype=torch.int32, device=gpu)
    cache.k_scales = torch.empty(pages, 8, 256, dtype=torch.float16, device=gpu)
    cache.v_scales = torch.empty(pages, 8, 256, dtype=torch.float16, device=gpu)
    table = torch.tensor([[65999, 3, 40000], [65001, 33000, -1]], dtype=torch.int32)
    for r in range(2):
        pos = torch.arange(small.lengths[r])
        cache.store(small.k[r].to(gpu), small.v[r].to(gpu), (table[r].long()[pos // 256] * 256 + pos % 256).to(gpu))
    q, _, lengths, _ = small.on_gpu()
    assert torch.equal(cache.attend(q, table.to(gpu), lengths), small.run())
    cu = torch.tensor([0, 600, 900], dtype=torch.int32, device=gpu)
    k, v = cache.load(table.to(gpu), cu, 900)
    assert torch.equal(k.cpu(), torch.cat([as_held(x)[0].half() for x in small.k]))
    assert torch.equal(v.cpu(), torch.cat([as_held(x)[0].half() for x in small.v]))


def test_same_result_every_time_streams_and_graphs(gpu):
    """eager, on another stream at the same time, and two captured graphs that are replayed in turn with eager calls between"""
    a = Problem(gpu, [3000, 20, 700], [1, 1, 1], 8, 2, 128, 128, 64, seed=1)
    b = Problem(gpu, [900, 5000], [1, 1], 8, 2, 128, 128, 64, seed=2)
    want = [x.run() for x in (a, b)]
    for _ in range(3):
        assert torch.equal(a.run(), want[0]) and torch.equal(b.run(), want[1])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    inputs = [x.on_gpu() for x in (a, b)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, x in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(x.cache.attend(inputs[i][0], inputs[i][1], inputs[i][2]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])
    graphs, outs = [], []
    for i, x in enumerate((a, b)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append([x.cache.attend(inputs[i][0], inputs[i][1], inputs[i][2]) for _ in range(2)])
        graphs.append(graph)
    for _ in range(4):
        for i in range(2):
            for o in outs[i]:
                o.zero_()
            graphs[i].replay()
        eager = a.run()
        torch.cuda.synchronize()
        assert torch.equal(eager, want[0]) and all(torch.equal(o, want[i]) for i in range(2) for o in outs[i])
    # replayed with other lengths: what the graph does follows the device's numbers
    inputs[0][2].copy_(torch.tensor([100, 15, 64], dtype=torch.int32))
    graphs[0].replay()
    a.lengths = [100, 15, 64]
    a.k, a.v = [k[:n] for k, n in zip(a.k, a.lengths)], [v[:n] for v, n in zip(a.v, a.lengths)]
    a.check(outs[0][0], 128 ** -0.5)


def test_refusals(gpu):
    p = Problem(gpu, [64, 30], [1, 1], 4, 2, 64, 40, 16)
    q, table, lengths, _ = p.on_gpu()
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=gpu)
    for args, kw, words in [
        ((q.float(), table, lengths), {}, "float16"), ((q.cpu(), table, lengths), {}, "GPU"), ((q, table.cpu(), lengths), {}, "GPU"),
        ((q[:, :3], table, lengths), {}, "multiple"), ((q[:, :, :32], table, lengths), {}, "wide"), ((q[:1], table, lengths), {}, "one row"),
        ((q, table.long(), lengths), {}, "table"), ((q, table[:, :0], lengths), {}, "column"), ((q, table, lengths[:1]), {}, "lengths"),
        ((q, table, lengths), dict(cu_q=cu[:2]), "cu_q"), ((q, table, lengths), dict(out=torch.empty(2, 4, 64, device=gpu).half()), "out"),
        ((q.permute(0, 2, 1).contiguous().permute(0, 2, 1), table, lengths), {}, "unit stride"),
    ]:
        with pytest.raises(RuntimeError, match=words):
            p.cache.attend(*args, **kw)
    k = torch.zeros(3, 2, 64, device=gpu).half()
    slots = torch.zeros(3, dtype=torch.int64, device=gpu)
    for args, words in [((k, k, slots), "wide"), ((k, k[:, :, :40], slots.int()), "slots"), ((k, k[:2, :, :40], slots), "per token"),
                        ((k[:, :1], k[:, :, :40], slots), "heads"), ((k, k[:, :, :40], slots.cpu()), "GPU"), ((k.bfloat16(), k[:, :, :40], slots), "float16")]:
        with pytest.raises(RuntimeError, match=words):
            p.cache.store(*args)
    for kw, words in [(dict(rows=-1), "rows"), (dict(cu=cu[:2]), "cu"), (dict(starts=cu), "starts"), (dict(k_out=k), "k_out")]:
        with pytest.raises(RuntimeError, match=words):
            p.cache.load(**{**dict(table=table, cu=cu, rows=5), **kw})
    from uniql_amd.quantize.quant_kv_cache import W4KVCache
    for bad in ((4, 24, 2, 64), (4, 16, 2, 129), (4, 16, 0, 64), (0, 16, 2, 64)):
        with pytest.raises(ValueError):
            W4KVCache(*bad, device=gpu)


def test_offsets_that_fall_leave_no_counts_behind(gpu):
    """requests whose rows are shared by several workgroups, with offsets that fall and rise again: the words that workgroups count their
    arrivals in are zeros afterwards, as every later call on the stream relies on"""
    from uniql_amd import ops
    p = Problem(gpu, [5000, 4000, 3000, 2000], [40, 30, 20, 10], 8, 1, 64, 64, 64)
    q, table, lengths, _ = p.on_gpu()
    for cu in ([0, 100, 0, 100, 0], [100, 0, 100, 0, 100], [50, 20, 90, 10, 100], [0, 2 ** 31 - 1, -5, 2 ** 31 - 1, 7]):
        p.cache.attend(q, table, lengths, cu_q=torch.tensor(cu, dtype=torch.int32, device=gpu))
        torch.cuda.synchronize()
        assert all(int(b.count_nonzero()) == 0 for b in ops._accum_cache.values())
    p.check(p.run(), 0.125)


@pytest.mark.parametrize("requests", [63, 64, 65, 130, 300])
@pytest.mark.parametrize("several", [False, True])
def test_many_requests(gpu, requests, several):
    """more requests than a wave has lanes; lengths from none to a few pages, some of them long"""
    gen = torch.Generator().manual_seed(requests)
    lengths = torch.randint(0, 60, (requests,), generator=gen).tolist()
    lengths[requests // 2], lengths[-1] = 900, 350
    tokens = torch.randint(0, 3, (requests,), generator=gen).tolist() if several else [1] * requests
    p = Problem(gpu, lengths, tokens, 4, 2, 32, 32, 16, seed=requests)
    p.check(p.run(), 32 ** -0.5)


@pytest.mark.parametrize("heads,kv_heads", [(5, 5), (6, 2), (9, 3), (64, 1), (80, 2)])
def test_heads_that_do_not_fill_four_waves(gpu, heads, kv_heads):
    p = Problem(gpu, [30, 700, 64, 1], [1, 1, 2, 1], heads, kv_heads, 64, 64, 16)
    p.check(p.run(), 0.125)


def test_a_scale_that_is_no_number_and_an_output_that_is_the_input(gpu):
    p = Problem(gpu, [64], [1], 4, 2, 64, 64, 16)
    q, table, lengths, _ = p.on_gpu()
    for scale in (float("nan"), float("inf"), 1e300):
        with pytest.raises(RuntimeError):
            p.cache.attend(q, table, lengths, scale=scale)
    with pytest.raises(RuntimeError, match="must not be q"):
        p.cache.attend(q, table, lengths, out=q)


@pytest.mark.parametrize("small,large", [(1e-4, 1e3), (1e-5, 6e4), (1.0, 6e4)])
@pytest.mark.parametrize("seen_first", [False, True])
def test_small_values_beside_large_ones_without_weight(gpu, small, large, seen_first):
    """nearly all weight is on one position whose values are tiny; others' are huge, but have no weight.  The result is that
    position's values to within the rounding of weights and results (half a step each) and of fp16 numbers below 2^-14 (2^-25)."""
    n, at = 400, 30 if seen_first else 370
    gen = torch.Generator().manual_seed(2)
    direction = torch.randn(64, generator=gen)
    k = torch.zeros(n, 1, 64).half()
    k[at, 0] = direction.half()

    def values(v):
        v = v * 0 + large * torch.sign(v)
        v[at] = (small * torch.randn(1, 64, generator=gen)).half()
        return v.half()

    p = Problem(gpu, [n], [1], 2, 1, 64, 64, 16, k_of=lambda _: k, v_of=values)
    p.q = (direction * 3).half().expand(1, 2, 64).contiguous()
    got = p.run(scale=1.0).cpu().double()[0, 0]      # one score of about 190, the others 0: weights of e^-190 and less
    want = as_held(p.v[0])[0][at, 0]
    assert ((got - want).abs() <= 2 ** -10 * want.abs() + 2 ** -25).all(), float((got - want).abs().max())


def test_graphs_of_one_stream_replayed_beside_each_other(gpu):
    """two graphs captured on a stream that has run eager calls, replayed on two other streams while that stream runs eager calls:
    each counts arrivals in words of its own"""
    from uniql_amd import ops
    problems = [Problem(gpu, [4000, 900], [1, 1], 8, 2, 128, 128, 64, seed=5 + i) for i in range(3)]
    inputs = [x.on_gpu()[:3] for x in problems]
    home = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(home):
        want = [x.cache.attend(*i) for x, i in zip(problems, inputs)]
    torch.cuda.synchronize()
    before = set(ops._accum_in_capture)
    graphs, outs = [], []
    for x, i in list(zip(problems, inputs))[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=home):
            outs.append([x.cache.attend(*i) for _ in range(3)])
        graphs.append(graph)
    words = [ops._accum_in_capture[key].data_ptr() for key in set(ops._accum_in_capture) - before]
    eager = ops._accum_cache[(home.device.index, home.cuda_stream)].data_ptr()
    assert len({eager, *words}) == 3
    others = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for out in outs:
            for o in out:
                o.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, others):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(home):
            got = [problems[2].cache.attend(*inputs[2]) for _ in range(3)]
        torch.cuda.synchronize()
        assert all(torch.equal(o, want[2]) for o in got)
        assert all(torch.equal(o, want[i]) for i in range(2) for o in outs[i])


def test_many_small_weights_beside_a_large_one(gpu):
    """one position has the weight 1 and the value -1, 60000 have 2^-24.3 and 1: together 0.0029, each below what is left of an fp16
    number scaled to 1.  Rounding: of the large weight 2^-11, of the small ones' sum (2^-24 of 2^-19.2) 6e-5, of the result 2^-12."""
    n = 60001
    k = torch.zeros(n, 1, 64).half()
    k[100, 0] = 1.0
    v = torch.ones(n, 1, 64).half()
    v[100] = -1.0
    p = Problem(gpu, [n], [1], 2, 1, 64, 64, 64, k_of=lambda _: k, v_of=lambda _: v)
    p.q = torch.ones(1, 2, 64).half()
    held_k, held_v = as_held(p.k[0])[0], as_held(p.v[0])[0]
    scale = 24.3 * 0.6931471805599453 / float(held_k[100, 0].sum())
    got = p.run(scale=scale).cpu().double()[0, 0]
    weight = 2.0 ** -24.3
    want = (held_v[100, 0] + (held_v[:, 0].sum(0) - held_v[100, 0]) * weight) / (1 + (n - 1) * weight)
    assert ((got - want).abs() <= 2 ** -10).all(), float((got - want).abs().max())


@pytest.mark.parametrize("lengths,tokens,h,g", [
    ([5000, 4000, 900, 300, 3000], [3000, 1, 700, 90, 2500], 2, 1),      # rows of two workgroups, of one, of a wave
    ([700] * 40 + [9000], [150] * 40 + [30], 4, 2), ([20000, 20000, 17], [1, 33, 5], 8, 1), ([12000], [12], 4, 4),
])
def test_scratch_of_just_the_size_asked_for(gpu, lengths, tokens, h, g):
    """many rows and few, shared and not: nothing in front of the scratch memory and behind it is written, the counts are zeros afterwards"""
    import ctypes
    from uniql_amd import _capi
    p = Problem(gpu, lengths, tokens, h, g, 32, 32, 64, seed=len(lengths))
    q, table, n, cu = p.on_gpu()
    c, lib, rows = p.cache, _capi.load(), p.q.shape[0]

    class Cache(ctypes.Structure):
        _fields_ = [(name, ctypes.c_void_p) for name in ("k_codes", "k_scales", "v_codes", "v_scales")] + \
                   [(name, ctypes.c_int) for name in ("pages", "page_size", "heads", "k_dim", "v_dim")]

    cache = Cache(c.k_codes.data_ptr(), c.k_scales.data_ptr(), c.v_codes.data_ptr(), c.v_scales.data_ptr(), c.num_pages, 64, g, 32, 32)
    acc, tmp = ctypes.c_size_t(0), ctypes.c_size_t(0)
    assert lib.uniql_kv4_attention_workspace(ctypes.byref(cache), rows, len(lengths), table.shape[1], h, ctypes.byref(acc), ctypes.byref(tmp)) == 0
    guard = 1 << 16
    accum = torch.full((acc.value + 2 * guard,), 77, dtype=torch.uint8, device=gpu)
    accum[guard:-guard] = 0
    temp = torch.full((tmp.value + 2 * guard,), 77, dtype=torch.uint8, device=gpu)
    out = torch.full((rows, h, 32), 9.0, device=gpu).half()
    torch.cuda.synchronize()
    for _ in range(2):
        code = lib.uniql_kv4_attention(q.data_ptr(), h * 32, 32, ctypes.byref(cache), table.data_ptr(), n.data_ptr(),
                                       None if cu is None else cu.data_ptr(), out.data_ptr(), h * 32, 32, accum[guard:].data_ptr(), acc.value,
                                       temp[guard:].data_ptr(), tmp.value, rows, len(lengths), table.shape[1], h, 32 ** -0.5,
                                       torch.cuda.current_stream().cuda_stream)
        assert code == 0
        torch.cuda.synchronize()
    assert (accum[guard:-guard] == 0).all()
    for t in (accum, temp):
        assert (t[:guard] == 77).all() and (t[-guard:] == 77).all()
    assert torch.equal(out, p.run())
    for r, (size, count) in enumerate(zip(lengths, tokens)):      # some rows of each request against 64 bits
        k, v = as_held(p.k[r])[0], as_held(p.v[r])
        for first in sorted({0, count // 2, max(0, count - 20)}):
            some = slice(p.cu[r] + first, p.cu[r] + min(count, first + 20))
            seen = size - count + first + 1
            o, mean_abs, spread = attention(p.q[some], k, v[0], 32 ** -0.5, seen)
            held = attention(p.q[some], k, v[1].unsqueeze(-1), 32 ** -0.5, seen)[0]
            assert ((out[some].cpu().double() - o).abs() <= bound(o, mean_abs, spread, size, held)).all(), (r, first)
