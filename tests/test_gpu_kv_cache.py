"""Pages and slots, writing the 4-bit cache and reading it back, against plain Python and 64-bit arithmetic."""
import numpy as np
import pytest
import torch

from tests.attention_reference import as_held

pytestmark = pytest.mark.gpu


# ---- pages and slots -------------------------------------------------------------------------------------------------
def assign_reference(new, lengths, table, free, page, most):
    """one request after the other"""
    columns = len(table[0]) if table else 1
    table, after, stack, memory = [list(r) for r in table], list(lengths), list(free), list(free)
    for r, n in enumerate(new):
        if n < 0:
            for p in table[r][:-(-lengths[r] // page)]:
                stack.append(p)
            after[r] = 0
    memory = list(stack)
    slots, positions, refused, cu, asked, available = [-1] * most, [0] * most, [0] * len(new), [0], 0, len(stack)
    total = 0
    for r, n in enumerate(new):
        begin = total
        total += max(n, 0)
        cu.append(min(total, most))
        if n <= 0:
            continue
        have, want = -(-lengths[r] // page), -(-(lengths[r] + n) // page)
        if lengths[r] + n > columns * page or total > most:
            refused[r] = 1
            continue
        asked += want - have
        if want > have and asked > available:
            refused[r] = 1
            continue
        for j in range(have, want):
            table[r][j] = stack.pop()
        for i in range(n):
            p = lengths[r] + i
            slots[begin + i], positions[begin + i] = table[r][p // page] * page + p % page, p
        after[r] = lengths[r] + n
    return slots, positions, refused, cu, after, len(stack), table, memory


def assign_problem(rng, rows, columns, page, cached, new_most, ended, pool_extra):
    lengths = [int(v) for v in rng.integers(0, min(cached, columns * page) + 1, rows)]
    new = [int(v) for v in rng.integers(0, new_most + 1, rows)]
    new = [-1 - int(rng.integers(0, 3)) if u < ended else n for n, u in zip(new, rng.random(rows))]
    held = [-(-n // page) for n in lengths]
    pool = sum(held) + pool_extra
    order = [int(v) for v in rng.permutation(pool)]
    table = [[-1] * columns for _ in range(rows)]
    for r, n in enumerate(held):
        for j in range(n):
            table[r][j] = order.pop()
    return lengths, new, table, order, pool


def run_assign(dev, new, lengths, table, free, pool, page, most, in_place):
    from uniql_amd import ops
    t = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    n, l, tab, count = t(new), t(lengths), t(table), t([len(free)])
    stack = t(list(free) + [-7] * (pool - len(free)))
    outs = {} if in_place else dict(lengths_out=torch.full_like(l, -5), count_out=torch.full_like(count, -5))
    slots, positions, cu, refused = ops.kv_assign_pages(n, l, tab, stack, count, page, most, **outs)
    l2, c2 = (l, count) if in_place else (outs["lengths_out"], outs["count_out"])
    if not in_place:
        assert l.tolist() == lengths and count.tolist() == [len(free)]
    assert n.tolist() == new
    return [x.tolist() for x in (slots, positions, refused, cu, l2, c2, tab, stack)]


@pytest.mark.parametrize("rows,columns,page,cached,new_most,ended,extra,cut", [
    (1, 1, 16, 0, 16, 0.0, 1, 0), (1, 8, 16, 100, 28, 0.0, 2, 0), (64, 12, 64, 700, 1, 0.0, 40, 0), (64, 12, 64, 700, 1, 0.0, 0, 0),
    (7, 40, 16, 300, 300, 0.3, 60, 5), (63, 5, 256, 1300, 200, 0.5, 0, 0), (300, 64, 16, 500, 400, 0.2, 1000, 0),
    (300, 64, 16, 500, 400, 0.2, 4000, -20000), (1024, 9, 32, 250, 3, 0.1, 100, 0), (1025, 9, 32, 250, 3, 0.1, 100, 3),
    (2500, 20, 16, 200, 40, 0.2, 1500, 0), (3, 4, 16, 60, 60, 0.0, 100, 0), (5, 2000, 16, 100, 30000, 0.0, 9000, 1),
])
@pytest.mark.parametrize("in_place", [True, False])
def test_assign(gpu, rows, columns, page, cached, new_most, ended, extra, cut, in_place):
    rng = np.random.default_rng(rows * 1000 + columns)
    lengths, new, table, free, pool = assign_problem(rng, rows, columns, page, cached, new_most, ended, extra)
    most = max(0, sum(max(n, 0) for n in new) + cut)
    got = run_assign(gpu, new, lengths, table, free, pool, page, most, in_place)
    slots, positions, refused, cu, after, count, tab, memory = assign_reference(new, lengths, table, free, page, most)
    assert got[3] == cu and got[2] == refused and got[4] == after and got[5] == [count]
    assert got[6] == tab
    assert got[7][:len(memory)] == memory and got[7][len(memory):] == [-7] * (pool - len(memory))
    assert got[0] == slots and got[1] == positions


def test_assign_without_requests_and_without_tokens(gpu):
    from uniql_amd import ops
    e = lambda *s: torch.zeros(*s, dtype=torch.int32, device=gpu)
    slots, positions, cu, refused = ops.kv_assign_pages(e(0), e(0), e(0, 3), e(4), e(1), 16, 5)
    assert slots.tolist() == [-1] * 5 and positions.tolist() == [0] * 5 and cu.tolist() == [0] and refused.tolist() == []
    slots, positions, cu, refused = ops.kv_assign_pages(e(2), e(2), e(2, 3), e(4), e(1), 16, 0)
    assert slots.numel() == 0 and cu.tolist() == [0, 0, 0] and refused.tolist() == [0, 0]


def test_assign_with_lengths_and_counts_that_cannot_be(gpu):
    """lengths below 0 or beyond the table's room, a count beyond the list: nothing outside the arrays is touched"""
    new, lengths = [1, 1, -1, -1, 4], [-3, 1000, -9, 10 ** 6, 3]
    got = run_assign(gpu, new, lengths, [[9, 9], [9, 9], [9, 9], [5, 6], [7, 8]], [], 6, 16, 6, False)
    assert got[2] == [1, 1, 0, 0, 0] and got[4] == [-3, 1000, 0, 0, 7] and got[5] == [2]
    assert got[0] == [-1, -1, 7 * 16 + 3, 7 * 16 + 4, 7 * 16 + 5, 7 * 16 + 6]


def test_assign_over_many_steps(gpu):
    """requests arrive, grow and end, in place, through the module; pages are never held twice"""
    from uniql_amd.quantize.quant_kv_cache import KVPages
    rng = np.random.default_rng(3)
    pages = KVPages(200, 16, 33, 30, device=gpu)
    lengths, free, table = [0] * 33, list(range(199, -1, -1)), [[-1] * 30 for _ in range(33)]
    for _ in range(60):
        new = [int(n) for n in rng.integers(0, 40, 33) * (rng.random(33) < 0.5)]
        new = [-1 if lengths[r] and rng.random() < 0.15 else n for r, n in enumerate(new)]
        most = sum(max(n, 0) for n in new)
        slots, positions, refused, cu, lengths, count, table, memory = assign_reference(new, lengths, table, free, 16, most)
        free = memory[:count]
        step = pages.assign(torch.tensor(new, dtype=torch.int32, device=gpu), most)
        assert step.slots.tolist() == slots and step.positions.tolist() == positions and step.refused.tolist() == refused
        assert pages.lengths.tolist() == lengths and pages.free_count.tolist() == [count] and pages.table.tolist() == table
        held = [p for r in range(33) for p in table[r][:-(-lengths[r] // 16)]]
        assert sorted(held + free) == list(range(200))


# ---- store and load ---------------------------------------------------------------------------------------------------
def new_cache(dev, pages, page, heads, d, e, fill=None):
    from uniql_amd.quantize.quant_kv_cache import W4KVCache
    c = W4KVCache(pages, page, heads, d, e, device=dev)
    if fill is not None:
        for t in (c.k_codes, c.v_codes):
            t.fill_(fill)
        for t in (c.k_scales, c.v_scales):
            t.fill_(3.0)
    return c


def fused_rows(gen, rows, heads, d, e, shift=0):
    """k and v as ranges of one buffer of rows, `shift` elements off its start"""
    buf = torch.randn(rows * (heads * (d + e) + shift) + shift, generator=gen).half()
    full = buf[shift:].view(rows, heads * (d + e) + shift)
    return buf, lambda b: (b[shift:].view(rows, -1)[:, :heads * d].view(rows, heads, d),
                           b[shift:].view(rows, -1)[:, heads * d:heads * (d + e)].view(rows, heads, e))


@pytest.mark.parametrize("tokens,heads,d,e,page", [(1, 1, 1, 1, 16), (1, 8, 128, 128, 64), (50, 2, 128, 64, 16), (33, 3, 108, 100, 32),
                                                   (7, 5, 33, 127, 128), (300, 8, 128, 128, 256), (19, 4, 2, 96, 16), (5, 7, 31, 32, 32)])
@pytest.mark.parametrize("shift", [0, 1, 8])
def test_store_then_load(gpu, tokens, heads, d, e, page, shift):
    gen = torch.Generator().manual_seed(tokens + d)
    buf, views = fused_rows(gen, tokens, heads, d, e, shift)
    k, v = views(buf)
    k[0, 0] = 0
    v[tokens // 2, heads - 1] *= 1e-4
    if tokens > 4:
        k[3] *= 300.0
        v[4, 0] = float("inf")
        k[2, 0, d // 2] = float("nan")
    pages = -(-tokens // page) + 2
    cache = new_cache(gpu, pages, page, heads, d, e)
    table = torch.randperm(pages, generator=gen).to(torch.int32)[None, :].contiguous()
    pos = torch.arange(tokens)
    slots = table[0].long()[pos // page] * page + pos % page
    gk, gv = views(buf.to(gpu))
    cache.store(gk, gv, slots.to(gpu))
    cu = torch.tensor([0, tokens], dtype=torch.int32, device=gpu)
    lk, lv = cache.load(table.to(gpu), cu, tokens)
    for got, x in ((lk, k), (lv, v)):
        want, _ = as_held(x)
        # the product of a code and a scale is exact in fp32 and rounded once
        assert torch.equal(got.cpu().isnan(), want.isnan())
        assert torch.equal(got.cpu().nan_to_num(), want.half().nan_to_num())


def test_codes_at_every_border_of_rounding(gpu):
    """x = (k + 1/2) s exactly, and its fp16 neighbours, for every mantissa of the scale: ties go to even, the rest to the nearest"""
    m = torch.arange(1024, 2048, dtype=torch.float64) / 1024
    for exponent in (-20, -14, -3, 4):
        top = (m * 2.0 ** exponent).half()
        s = (top.double() * 2 / 15).half().double()
        rows = torch.zeros(1024, 1, 64, dtype=torch.float16)
        rows[:, 0, 0] = top
        at = 1
        for i in range(-7, 7):
            mid = ((i + 0.5) * s).half()
            for x in (mid, torch.nextafter(mid.float(), torch.tensor(9e4)).half(), (mid.view(torch.int16) + 1).view(torch.float16),
                      (mid.view(torch.int16) - 1).view(torch.float16)):
                if at < 64:
                    rows[:, 0, at] = torch.where(x.abs() <= top, x, torch.zeros_like(x))
                    at += 1
        cache = new_cache(gpu, 4, 256, 1, 64, 64)
        table = torch.arange(4, dtype=torch.int32, device=gpu)[None]
        cache.store(rows.to(gpu), rows.flip(2).contiguous().to(gpu), torch.arange(1024, device=gpu))
        k, v = cache.load(table, torch.tensor([0, 1024], dtype=torch.int32, device=gpu), 1024)
        want = as_held(rows)[0].half()
        assert torch.equal(k.cpu(), want) and torch.equal(v.cpu(), want.flip(2))


def test_store_leaves_out_places_outside_the_pool(gpu):
    cache = new_cache(gpu, 2, 16, 2, 40, 40, fill=0x13579bdf)
    before = [t.clone() for t in cache.buffers()]
    x = torch.randn(4, 2, 40, device=gpu).half()
    cache.store(x, x, torch.tensor([-1, 32, 10 ** 12, -2 ** 62], device=gpu))
    assert all(torch.equal(a, b) for a, b in zip(before, cache.buffers()))
    cache.store(x, x, torch.tensor([-1, 31, 32, 0], device=gpu))
    changed = (before[1] != cache.k_scales).any(1).nonzero().tolist()
    assert changed == [[0, 0], [1, 15]]
    cache.store(x[:0], x[:0], torch.zeros(0, dtype=torch.int64, device=gpu))


def test_load_of_requests_and_what_is_left_alone(gpu):
    """starts, empty requests, rows in front of the first and behind the last, page numbers and positions that do not exist"""
    gen = torch.Generator().manual_seed(5)
    cache = new_cache(gpu, 6, 16, 3, 50, 20)
    k, v = torch.randn(96, 3, 50, generator=gen).half(), torch.randn(96, 3, 20, generator=gen).half()
    cache.store(k.to(gpu), v.to(gpu), torch.arange(96, device=gpu))
    table = torch.tensor([[3, 1], [5, 99], [0, -1], [2, 4]], dtype=torch.int32, device=gpu)
    cu = torch.tensor([2, 8, 8, 30, 40], dtype=torch.int32, device=gpu)
    starts = torch.tensor([13, 0, 12, 28], dtype=torch.int32, device=gpu)
    k_out, v_out = torch.full((45, 3, 50), 7.0, device=gpu).half(), torch.full((45, 3, 20), 7.0, device=gpu).half()
    got = cache.load(table, cu, 45, starts=starts, k_out=k_out, v_out=v_out)
    assert got[0] is not None and got[0].data_ptr() == k_out.data_ptr()
    for out, x in ((k_out.cpu(), k), (v_out.cpu(), v)):
        held = as_held(x)[0].half()
        assert (out[:2] == 7).all() and (out[40:] == 7).all()
        assert torch.equal(out[2:5], held[48 + 13:64]) and torch.equal(out[5:8], held[16:19])
        assert torch.equal(out[8:12], held[12:16]) and out[12:30].isnan().all()
        assert torch.equal(out[30:34], held[4 * 16 + 12:4 * 16 + 16])
        assert out[34:40].isnan().all()   # positions 32 and more: the table has no such column


def test_store_captured_and_replayed(gpu):
    cache, eager = new_cache(gpu, 4, 16, 2, 128, 128), new_cache(gpu, 4, 16, 2, 128, 128)
    x = torch.randn(9, 2, 128, device=gpu).half()
    slots = torch.randperm(64, device=gpu)[:9]
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        cache.store(x, x, slots)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        cache.store(x, x, slots)
    for _ in range(4):
        x.copy_(torch.randn_like(x))
        slots.copy_(torch.randperm(64, device=gpu)[:9])
        torch.cuda.synchronize()
        graph.replay()
        eager.store(x, x, slots)
        torch.cuda.synchronize()
        for name in ("k_codes", "k_scales", "v_codes", "v_scales"):
            a, b = getattr(cache, name), getattr(eager, name)
            for s in slots.tolist():
                if name == "v_codes":
                    assert torch.equal(a[s // 16, :, s % 16 // 4, :, s % 4], b[s // 16, :, s % 16 // 4, :, s % 4])
                else:
                    assert torch.equal(a[s // 16, :, s % 16], b[s // 16, :, s % 16])


def test_a_cache_whose_tensors_are_replaced_or_copied(gpu):
    """calls follow the module's own tensors: after an assignment, a move, a copy"""
    import copy
    import pickle
    x = torch.randn(20, 2, 40, generator=torch.Generator().manual_seed(1)).half()
    slots, table = torch.arange(20, device=gpu), torch.arange(2, dtype=torch.int32, device=gpu)[None]
    cu = torch.tensor([0, 20], dtype=torch.int32, device=gpu)
    want = as_held(x)[0].half()
    cache = new_cache(gpu, 2, 16, 2, 40, 40)
    cache.store(x.to(gpu), x.to(gpu), slots)
    other = copy.deepcopy(cache)
    third = pickle.loads(pickle.dumps(cache))
    old = cache.k_scales
    cache.k_scales = torch.zeros_like(old)
    assert (cache.load(table, cu, 20)[0] == 0).all() and torch.equal(cache.load(table, cu, 20)[1].cpu(), want)
    cache.k_scales = old
    moved = cache.cpu().to(gpu)
    for c in (cache, other, third, moved):
        k, v = c.load(table, cu, 20)
        assert torch.equal(k.cpu(), want) and torch.equal(v.cpu(), want)
    other.store(torch.zeros_like(x).to(gpu), torch.zeros_like(x).to(gpu), slots)
    assert (other.load(table, cu, 20)[0] == 0).all() and torch.equal(cache.load(table, cu, 20)[0].cpu(), want)


def test_a_request_without_need_behind_one_that_is_refused(gpu):
    """it is served, and takes nothing: the pages that the refused one asked for in vain stay free"""
    got = run_assign(gpu, [40, 1, 20, 3], [0, 5, 0, 10], [[-1] * 4, [7, -1, -1, -1], [-1] * 4, [8, -1, -1, -1]], [4, 6], 10, 16, 64, True)
    slots, positions, refused, cu, after, count, tab, memory = assign_reference(
        [40, 1, 20, 3], [0, 5, 0, 10], [[-1] * 4, [7, -1, -1, -1], [-1] * 4, [8, -1, -1, -1]], [4, 6], 16, 64)
    assert refused == [1, 0, 1, 0] and count == 2
    assert [got[2], got[4], got[5], got[0], got[6]] == [refused, after, [count], slots, tab]


def test_a_cache_whose_tensors_are_replaced_past_its_attributes(gpu):
    """register_buffer, a write to the module's dict of buffers, a functional call: store, load and attend take the tensors that are there"""
    gen = torch.Generator().manual_seed(3)
    a, b = torch.randn(20, 2, 40, generator=gen).half(), torch.randn(20, 2, 40, generator=gen).half()
    slots, table = torch.arange(20, device=gpu), torch.arange(2, dtype=torch.int32, device=gpu)[None]
    cu, lengths = torch.tensor([0, 20], dtype=torch.int32, device=gpu), torch.tensor([20], dtype=torch.int32, device=gpu)
    q = torch.randn(1, 4, 40, generator=gen).half().to(gpu)
    names = ("k_codes", "k_scales", "v_codes", "v_scales")
    other = new_cache(gpu, 2, 16, 2, 40, 40)
    other.store(b.to(gpu), b.to(gpu), slots)
    want = other.attend(q, table, lengths)

    def fresh():
        cache = new_cache(gpu, 2, 16, 2, 40, 40)
        cache.store(a.to(gpu), a.to(gpu), slots)
        return cache

    def is_other(cache):
        return torch.equal(cache.load(table, cu, 20)[0].cpu(), as_held(b)[0].half()) and torch.equal(cache.attend(q, table, lengths), want)

    cache = fresh()
    for name in names:
        cache.register_buffer(name, getattr(other, name).clone(), persistent=False)
    assert is_other(cache)
    cache = fresh()
    mine = [t.clone() for t in cache.buffers()]
    for name in names:
        cache._buffers[name] = torch.zeros_like(getattr(other, name))
    cache.store(b.to(gpu), b.to(gpu), slots)
    assert is_other(cache)

    class Call(torch.nn.Module):
        def __init__(self, cache):
            super().__init__()
            self.cache = cache

        def forward(self):
            return is_other(self.cache)

    cache = fresh()
    assert not Call(cache)()
    assert torch.func.functional_call(Call(cache), {"cache." + name: getattr(other, name) for name in names}, ())
    assert not Call(cache)() and all(torch.equal(x, y) for x, y in zip(mine, cache.buffers()))


def test_a_full_list_of_as_many_pages_as_numbers_go(gpu):
    """2^31 - 1 free pages, as many as the list has room for, and a request that gives back another hundred: nothing is written"""
    from uniql_amd import ops
    pool = 2 ** 31 - 1
    t = lambda v: torch.tensor(v, dtype=torch.int32, device=gpu)
    free = torch.full((pool,), -7, dtype=torch.int32, device=gpu)
    for count, kept in ((pool, 0), (pool - 60, 60)):
        n = t([count])
        ops.kv_assign_pages(t([-1]), t([1600]), torch.arange(100, dtype=torch.int32, device=gpu)[None], free, n, 16, 4)
        assert n.tolist() == [pool] and free[count:].tolist() == list(range(kept))
        assert int(free[:count].amax()) == -7 and int(free[:count].amin()) == -7


def test_assign_refuses_arrays_that_share_memory(gpu):
    """what the call writes is no part of what it reads or writes otherwise; lengths and the count may be replaced in place"""
    from uniql_amd import ops
    words = torch.zeros(200, dtype=torch.int32, device=gpu)
    new, lengths, count, table, free = words[:4], words[4:8], words[8:9], words[9:49].view(4, 10), words[49:69]
    spare, one = words[69:73], words[73:74]

    def call(**kw):
        a = {**dict(new=new, lengths=lengths, table=table, free=free, count=count, lengths_out=spare, count_out=one), **kw}
        return ops.kv_assign_pages(a["new"], a["lengths"], a["table"], a["free"], a["count"], 16, 8, lengths_out=a["lengths_out"],
                                   count_out=a["count_out"])

    call(), call(lengths_out=None, count_out=None), call(lengths_out=lengths, count_out=count), call(lengths=words[1:5])
    for kw in (dict(lengths_out=new), dict(lengths_out=words[2:6]), dict(lengths_out=words[5:9]), dict(lengths_out=words[6:10]),
               dict(lengths_out=words[40:44]), dict(lengths_out=words[66:70]), dict(count_out=words[3:4]), dict(count_out=words[5:6]),
               dict(count_out=words[70:71]), dict(count_out=words[30:31]), dict(count_out=words[60:61]), dict(free=words[48:60]),
               dict(free=words[5:20]), dict(table=words[2:42].view(4, 10)), dict(table=words[30:70].view(4, 10)), dict(new=words[45:49]),
               dict(lengths=words[50:54]), dict(count=words[50:51]), dict(new=lengths, lengths_out=None), dict(count=words[5:6], lengths_out=None)):
        with pytest.raises(RuntimeError, match="share memory"):
            call(**kw)
    assert int(words.count_nonzero()) == 0
