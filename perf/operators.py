"""The attention side of a decoder layer behind the 4-bit projections: what is timed, and what its results are.

A case is a dict of plain values whose "kind" names one operator:

    assign   block tables and slot maps: requests that arrive, grow by some tokens or end take pages from a free list
             and give them back, and every new token gets its place in the paged cache
    store    keys and values of new tokens go into the paged 4-bit cache, and are read back from it as fp16, the way
             a prompt that is taken in pieces has its earlier pieces ready for the next one
    attend   attention of each request's newest tokens over its pages of the 4-bit cache (grouped heads, causal)
    prompt   causal attention over the whole prompts of several requests that lie behind each other without padding

The cache holds a vector x of one token and one key / value head as s (c - 8) with s = fp16(max|x| 2/15) and
c = clamp(round(x / s) + 8, 0, 15): the arithmetic of the 4-bit projections, one scale for the vector.

listed() holds the sizes looked at first, draw() gives others of the same ranges.  Head counts and widths are those of
Llama-3.1-8B (32 and 8 heads of 128), Llama-2-7B (32 and 32) and Qwen2-7B (28 and 4), whole and pruned.
"""
from __future__ import annotations

import math

import torch

own = False
DEVICE = "cuda:0"


# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # one step of a serving loop: 64 requests advance by a token, a few of them need a new page
        dict(name="assign_64_by_1", kind="assign", requests=64, cached=700, tokens=1, released=0.0, page=64, spare=1.0),
        # the scheduler's largest step: hundreds of requests, prompts among single tokens, some end, the last find no page
        dict(name="assign_500_mixed", kind="assign", requests=500, cached=900, tokens=250, released=0.15, page=16, spare=0.9),
        # the keys and values of one step of 48 requests
        dict(name="store_48x1", kind="store", requests=48, cached=600, tokens=1, kv_heads=8, head_dim=128, v_dim=128, page=64),
        # pieces of odd length of a pruned model's prompts, rows of the fused projection's output
        dict(name="store_7x111_pruned", kind="store", requests=7, cached=333, tokens=111, kv_heads=32, head_dim=108, v_dim=100, page=32),
        # a long prompt
        dict(name="store_1x16384", kind="store", requests=1, cached=0, tokens=16384, kv_heads=8, head_dim=128, v_dim=128, page=256),
        # one user, one token, a chat of some length: latency
        dict(name="attend_1x4096", kind="attend", requests=1, context=4096, ragged=False, tokens=1, heads=32, kv_heads=8,
             head_dim=128, v_dim=128, page=64),
        # continuous batching: requests of very different lengths advance together
        dict(name="attend_48_ragged", kind="attend", requests=48, context=8192, ragged=True, tokens=1, heads=32, kv_heads=8,
             head_dim=128, v_dim=128, page=16),
        # a pruned model without grouped heads, five drafted tokens to verify for each request
        dict(name="attend_9x5_pruned", kind="attend", requests=9, context=2049, ragged=True, tokens=5, heads=32, kv_heads=32,
             head_dim=108, v_dim=100, page=32),
        # long documents: what the cache's bandwidth allows
        dict(name="attend_16x65536", kind="attend", requests=16, context=65536, ragged=False, tokens=1, heads=32, kv_heads=8,
             head_dim=128, v_dim=128, page=256),
        # a short prompt of odd length on a pruned model: time to first token
        dict(name="prompt_333_pruned", kind="prompt", sequences=1, tokens=333, ragged=False, heads=32, kv_heads=8, head_dim=108,
             v_dim=108),
        # a scheduler's batch of prompts of very different lengths
        dict(name="prompt_24_packed", kind="prompt", sequences=24, tokens=1500, ragged=True, heads=32, kv_heads=8, head_dim=128,
             v_dim=128),
        # a long document: the largest call
        dict(name="prompt_16384", kind="prompt", sequences=1, tokens=16384, ragged=False, heads=32, kv_heads=8, head_dim=128,
             v_dim=128),
    ]


def _spread(rng, low, high):
    """a whole number whose logarithm is uniform"""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _head(rng):
    """a head width: the models' own ones or any even width a pruned model may have"""
    return rng.choice((64, 96, 128, 2 * rng.randint(16, 64), 2 * rng.randint(16, 64)))


def draw(rng):
    kind = rng.choice(("assign", "store", "attend", "prompt"))
    heads, kv_heads = rng.choice(((32, 8), (32, 32), (28, 4)))
    head_dim = _head(rng)
    v_dim = head_dim if rng.random() < 0.6 else _head(rng)
    page = rng.choice((16, 32, 64, 128, 256))
    if kind == "assign":
        requests = _spread(rng, 1, 600)
        return dict(kind=kind, requests=requests, cached=_spread(rng, 1, 4000), tokens=_spread(rng, 1, 125000 // requests),
                    released=rng.choice((0.0, rng.uniform(0.0, 0.5))), page=page, spare=rng.uniform(0.5, 1.5))
    if kind == "store":
        requests = _spread(rng, 1, 64)
        tokens = _spread(rng, 1, 16384 * 8 // (kv_heads * requests))
        return dict(kind=kind, requests=requests, cached=_spread(rng, 1, 1000), tokens=tokens, kv_heads=kv_heads, head_dim=head_dim,
                    v_dim=v_dim, page=page)
    if kind == "attend":
        requests = _spread(rng, 1, 64)
        context = _spread(rng, 1, min(65536, 16 * 65536 * 8 // (kv_heads * requests)))
        return dict(kind=kind, requests=requests, context=context, ragged=rng.random() < 0.7,
                    tokens=rng.choice((1, 1, 1, rng.randint(2, 8))), heads=heads, kv_heads=kv_heads, head_dim=head_dim, v_dim=v_dim,
                    page=page)
    sequences = _spread(rng, 1, 64)
    return dict(kind=kind, sequences=sequences, tokens=_spread(rng, 1, int(16384 / math.sqrt(sequences) / 1.5)),
                ragged=rng.random() < 0.7, heads=heads, kv_heads=kv_heads, head_dim=head_dim, v_dim=v_dim)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _rng(seed):
    return torch.Generator(DEVICE).manual_seed(seed * 7919 + 17), torch.Generator().manual_seed(seed * 104729 + 5)


def _lengths(gen, count, most, ragged):
    """lengths of `count` requests: all `most`, or from a token to `most` with short ones more frequent"""
    if not ragged:
        return [most] * count
    return [int(v) for v in (most ** torch.rand(count, generator=gen, dtype=torch.float64)).round().clamp(1, most)]


def _requests(case):
    """(tokens in the cache, new tokens) of each request: the case's own; a seed only orders them.  -1 new tokens: it ends"""
    kind = case["kind"]
    gen = torch.Generator().manual_seed(sum(ord(c) * 31 ** (i % 7) for i, c in enumerate(repr(sorted((k, v) for k, v in case.items() if k != "name")))))
    if kind == "assign":
        n = case["requests"]
        cached = _lengths(gen, n, case["cached"], True)
        new = [1] * n if case["tokens"] == 1 else _lengths(gen, n, 2 * case["tokens"], True)
        new = [-1 if u < case["released"] else t for t, u in zip(new, torch.rand(n, generator=gen).tolist())]
        if n > 4:
            cached[: n // 8] = [0] * (n // 8)   # rows without a request so far
        return list(zip(cached, new))
    if kind == "store":
        n = case["requests"]
        cached = _lengths(gen, n, case["cached"], True) if case["cached"] else [0] * n
        return list(zip(cached, _lengths(gen, n, case["tokens"], n > 1 and case["tokens"] > 1)))
    if kind == "attend":
        lengths = _lengths(gen, case["requests"], case["context"], case["ragged"])
        lengths[0] = case["context"]
        return [(max(n - case["tokens"], 0), case["tokens"]) for n in lengths]
    return [(0, n) for n in _lengths(gen, case["sequences"], int(case["tokens"] * 1.5) if case["ragged"] else case["tokens"], case["ragged"])]


def _in_order(case, gen):
    pairs = _requests(case)
    pairs = [pairs[i] for i in torch.randperm(len(pairs), generator=gen).tolist()]
    return [a for a, _ in pairs], [b for _, b in pairs]


def _offsets(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _vectors(gen, rows, heads, width):
    """activations as projections give them: a few channels are several times larger than the others"""
    x = torch.randn(rows, heads, width, generator=gen, device=DEVICE)
    x[:, :, :: 37] *= 4.0
    return x.half()


def _fused(gen, rows, kv_heads, head_dim, v_dim, heads=0):
    """q, k and v as the column ranges of the fused projection's output; without heads only k and v"""
    widths = [heads * head_dim, kv_heads * head_dim, kv_heads * v_dim]
    buffer = torch.empty(rows, sum(widths), dtype=torch.float16, device=DEVICE)
    q, k, v = buffer.split(widths, dim=1)
    q, k, v = q.view(rows, heads, head_dim) if heads else None, k.view(rows, kv_heads, head_dim), v.view(rows, kv_heads, v_dim)
    if heads:
        q.copy_(torch.randn(rows, heads, head_dim, generator=gen, device=DEVICE) * 1.5)
    k.copy_(_vectors(gen, rows, kv_heads, head_dim))
    v.copy_(_vectors(gen, rows, kv_heads, v_dim))
    return q, k, v


def _pages_of(lengths, page):
    return [(n + page - 1) // page for n in lengths]


def _table(gen, lengths, page):
    """a table of pages in no order at all, and how many pages there are"""
    need = _pages_of(lengths, page)
    total = sum(need) + 3
    order = torch.randperm(total, generator=gen).to(torch.int32)
    table = torch.full((len(lengths), max(need + [1])), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        at += n
    return table, total


def _assign_inputs(case, seed):
    _, gen = _rng(seed)
    page = case["page"]
    lengths, new = _in_order(case, gen)
    n = len(new)
    lengths, new = torch.tensor(lengths, dtype=torch.int32), torch.tensor(new, dtype=torch.int32)
    table, taken = _table(gen, lengths.tolist(), page)
    held = sum(_pages_of(lengths.tolist(), page))
    grown = [a + max(b, 0) for a, b in zip(lengths.tolist(), new.tolist())]
    need = sum(_pages_of(grown, page)) - held
    free = max(int(need * case["spare"]) + (2 if case["spare"] >= 1 else 0), 1)
    columns = max(_pages_of(grown, page) + [1])
    wide = torch.full((n, columns), -1, dtype=torch.int32)
    wide[:, : min(table.shape[1], columns)] = table[:, :columns]
    pool = taken + free
    used = torch.zeros(pool, dtype=torch.bool)
    used[wide[wide >= 0].long()] = True
    order = torch.randperm(pool, generator=gen)
    stack = order[~used[order]].to(torch.int32)[:free]
    free_pages = torch.full((pool,), -1, dtype=torch.int32)
    free_pages[: stack.numel()] = stack
    most = int(new.clamp_min(0).sum()) + n % 5   # a batch padded by a few tokens
    count = torch.tensor([stack.numel()], dtype=torch.int32)
    return new, lengths, wide, free_pages, count, most


def _slots_of(table, lengths, starts, page):
    """where the positions starts[r] .. lengths[r] of each request lie"""
    out = []
    for r, (a, b) in enumerate(zip(starts, lengths)):
        pos = torch.arange(a, b)
        out.append(table[r].long()[pos // page] * page + pos % page)
    return torch.cat(out)


def _store_inputs(case, seed):
    gpu, gen = _rng(seed)
    cached, new = _in_order(case, gen)
    lengths = [a + b for a, b in zip(cached, new)]
    table, pages = _table(gen, lengths, case["page"])
    slots = _slots_of(table, lengths, cached, case["page"])
    _, k, v = _fused(gpu, sum(new), case["kv_heads"], case["head_dim"], case["v_dim"])
    return k, v, slots, table, pages, cached, _offsets(new)


def _attend_inputs(case, seed):
    """q, table, lengths, first row of each request, and a function that gives a request's keys and values"""
    gpu, gen = _rng(seed)
    n, tokens = case["requests"], case["tokens"]
    lengths = [a + b for a, b in zip(*_in_order(case, gen))]
    table, pages = _table(gen, lengths, case["page"])
    q = (torch.randn(n * tokens, case["heads"], case["head_dim"], generator=gpu, device=DEVICE) * 1.5).half()

    def keys_values(r):
        g = torch.Generator(DEVICE).manual_seed(seed * 1000003 + r)
        return _vectors(g, lengths[r], case["kv_heads"], case["head_dim"]), _vectors(g, lengths[r], case["kv_heads"], case["v_dim"])

    return q, table, pages, lengths, keys_values


def _prompt_inputs(case, seed):
    gpu, gen = _rng(seed)
    _, lengths = _in_order(case, gen)
    q, k, v = _fused(gpu, sum(lengths), case["kv_heads"], case["head_dim"], case["v_dim"], case["heads"])
    return q, k, v, _offsets(lengths)


def prepare(case, seed):
    kind = case["kind"]
    state = dict(case)
    if kind == "assign":
        new, lengths, table, free_pages, count, most = _assign_inputs(case, seed)
        state.update(new=new.to(DEVICE), lengths=lengths.to(DEVICE), table=table.to(DEVICE), free_pages=free_pages.to(DEVICE),
                     count=count.to(DEVICE), most=most)
        # the state of the step before is kept, as a program does that may take a step back
        state.update(lengths_out=torch.empty_like(state["lengths"]), count_out=torch.empty_like(state["count"]))
        return state
    if kind == "store":
        k, v, slots, table, pages, cached, cu = _store_inputs(case, seed)
        state.update(k=k, v=v, slots=slots.to(DEVICE), table=table.to(DEVICE), total=cu[-1],
                     starts=torch.tensor(cached, dtype=torch.int32, device=DEVICE), cu=torch.tensor(cu, dtype=torch.int32, device=DEVICE))
        state["cache"] = _new_cache(case, pages)
        return state
    if kind == "attend":
        q, table, pages, lengths, keys_values = _attend_inputs(case, seed)
        state.update(q=q, table=table.to(DEVICE), host_lengths=lengths, lengths=torch.tensor(lengths, dtype=torch.int32, device=DEVICE),
                     scale=case["head_dim"] ** -0.5)
        tokens = case["tokens"]
        state["cu"] = None if tokens == 1 else torch.arange(0, (case["requests"] + 1) * tokens, tokens, dtype=torch.int32, device=DEVICE)
        cache = state["cache"] = _new_cache(case, pages)
        for r, n in enumerate(lengths):
            k, v = keys_values(r)
            slots = _slots_of(table[r:r + 1], [n], [0], case["page"]).to(DEVICE)
            if own:
                cache.store(k, v, slots)
            else:
                _plain_store(cache, k, v, slots)
        return state
    q, k, v, cu = _prompt_inputs(case, seed)
    state.update(q=q, k=k, v=v, host_cu=cu, cu=torch.tensor(cu, dtype=torch.int32, device=DEVICE), scale=case["head_dim"] ** -0.5)
    return state


def _new_cache(case, pages):
    if own:
        from uniql_amd.quantize.quant_kv_cache import W4KVCache
        return W4KVCache(pages, case["page"], case["kv_heads"], case["head_dim"], case["v_dim"], device=DEVICE)
    places = pages * case["page"]
    return dict(k=torch.zeros(places, case["kv_heads"], case["head_dim"], dtype=torch.int8, device=DEVICE),
                v=torch.zeros(places, case["kv_heads"], case["v_dim"], dtype=torch.int8, device=DEVICE),
                ks=torch.zeros(places, case["kv_heads"], dtype=torch.float16, device=DEVICE),
                vs=torch.zeros(places, case["kv_heads"], dtype=torch.float16, device=DEVICE))


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    kind = s["kind"]
    if kind == "assign":
        from uniql_amd import ops
        slots, positions, cu, refused = ops.kv_assign_pages(s["new"], s["lengths"], s["table"], s["free_pages"], s["count"], s["page"],
                                                            s["most"], lengths_out=s["lengths_out"], count_out=s["count_out"])
        return dict(slots=slots, positions=positions, cu=cu, refused=refused, lengths=s["lengths_out"], count=s["count_out"],
                    table=s["table"], free_pages=s["free_pages"])
    if kind == "store":
        s["cache"].store(s["k"], s["v"], s["slots"])
        k, v = s["cache"].load(s["table"], s["cu"], s["total"], starts=s["starts"])
        return dict(k=k, v=v)
    if kind == "attend":
        return s["cache"].attend(s["q"], s["table"], s["lengths"], cu_q=s["cu"], scale=s["scale"])
    from uniql_amd.attention import prompt_attention
    return prompt_attention(s["q"], s["k"], s["v"], s["cu"], scale=s["scale"])


def _run_plain(s):
    return {"assign": _plain_assign, "store": _plain_store_load, "attend": _plain_attend, "prompt": _plain_prompt}[s["kind"]](s)


def _plain_assign(s):
    new, lengths, table, free_pages, page, most = s["new"], s["lengths"].long(), s["table"], s["free_pages"], s["page"], s["most"]
    rows, columns = table.shape
    ends, begins = new.lt(0), new.clamp_min(0).long()
    held = (lengths + page - 1) // page
    # pages of ended requests go on top of the free list, request after request
    column = torch.arange(columns, device=table.device)
    back = table[(column < held[:, None]) & ends[:, None]]
    count = s["count"].long()
    place = count + torch.arange(back.numel(), device=table.device)
    free_pages[place] = back
    count = count + back.numel()
    # requests in order take what they need from the top
    upto = torch.cumsum(begins, 0)
    fits = (begins > 0) & (lengths + begins <= columns * page) & (upto <= most)
    need = torch.where(fits, (lengths + begins + page - 1) // page - held, torch.zeros_like(held))
    taken = torch.cumsum(need, 0)
    served = fits & ((need == 0) | (taken <= count))
    first = taken - need
    fills = (column >= held[:, None]) & (column < (held + need)[:, None]) & served[:, None]
    source = (count - 1 - first)[:, None] - (column - held[:, None])
    table.copy_(torch.where(fills, free_pages[source.clamp(0, free_pages.numel() - 1)], table))
    s["count_out"].copy_(count - torch.where(served, taken, torch.zeros_like(taken)).amax())
    s["lengths_out"].copy_(torch.where(ends, torch.zeros_like(lengths), torch.where(served, lengths + begins, lengths)))
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device=table.device), upto]).clamp_max(most)
    token = torch.arange(most, device=table.device)
    request = torch.searchsorted(cu, token, right=True) - 1
    there = (request < rows) & served[request.clamp_max(rows - 1)]
    request = request.clamp_max(rows - 1)
    position = torch.where(there, lengths[request] + token - cu[request], torch.zeros_like(token))
    slot = table[request, position // page].long() * page + position % page
    return dict(slots=torch.where(there, slot, torch.full_like(slot, -1)), positions=position.int(), cu=cu.int(),
                refused=((begins > 0) & ~served).int(), lengths=s["lengths_out"], count=s["count_out"], table=table, free_pages=free_pages)


def _quantise(x):
    """codes (c - 8) and scales of the vectors along the last axis; 64 bits next to the borders of rounding"""
    x = x.double()
    s = (x.abs().amax(-1) * 2.0 / 15.0).half()
    c = torch.where(s[..., None] > 0, torch.round(x / s[..., None].double()), torch.zeros_like(x)).clamp(-8, 7)
    return c.to(torch.int8), s


def _plain_store(cache, k, v, slots):
    for name, x in (("k", k), ("v", v)):
        c, s = _quantise(x)
        cache[name][slots] = c
        cache[name + "s"][slots] = s


def _plain_store_load(s):
    cache, page = s["cache"], s["page"]
    _plain_store(cache, s["k"], s["v"], s["slots"])
    cu, token = s["cu"].long(), torch.arange(s["total"], device=DEVICE)
    request = torch.searchsorted(cu, token, right=True) - 1
    position = s["starts"].long()[request] + token - cu[request]
    at = s["table"][request, position // page].long() * page + position % page
    return dict(k=(cache["k"][at].float() * cache["ks"][at].float()[..., None]).half(),
                v=(cache["v"][at].float() * cache["vs"][at].float()[..., None]).half())


def _softmax_product(q, k, v, scale, first_limit):
    """softmax(scale q k^T) v for one sequence: q [t, h, d], k [n, g, d], v [n, g, e] in 32 bits; row i sees the first
    first_limit + i keys; rows are taken in pieces that keep the scores below 2 GB"""
    t, h, d = q.shape
    n, g, e = v.shape
    out = torch.zeros(t, h, e, device=q.device)
    kt, vt = k.permute(1, 2, 0).contiguous(), v.permute(1, 0, 2).contiguous()
    piece = max(1, min(t, (1 << 29) // (h * n)))
    for at in range(0, t, piece):
        rows = q[at:at + piece]
        m = rows.shape[0]
        folded = rows.reshape(m, g, h // g, d).permute(1, 2, 0, 3).reshape(g, h // g * m, d)
        score = torch.matmul(folded * scale, kt).view(g, h // g, m, n)
        hidden = torch.arange(n, device=q.device) >= first_limit + at + torch.arange(m, device=q.device)[:, None]
        score.masked_fill_(hidden, -math.inf)
        top = score.amax(-1, keepdim=True).clamp_min(-3.0e38)
        p = torch.exp_(score.sub_(top))
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p.view(g, h // g * m, n), vt).view(g, h // g, m, e) / total.clamp_min(1e-38)
        out[at:at + m] = o.permute(2, 0, 1, 3).reshape(m, h, e)
    return out


def _plain_attend(s):
    cache, page, tokens = s["cache"], s["page"], s["tokens"]
    out = torch.empty(s["q"].shape[0], s["heads"], s["v_dim"], dtype=torch.float16, device=DEVICE)
    for r, n in enumerate(s["host_lengths"]):
        position = torch.arange(n, device=DEVICE)
        at = s["table"][r].long()[position // page] * page + position % page
        k = cache["k"][at].float() * cache["ks"][at].float()[..., None]
        v = cache["v"][at].float() * cache["vs"][at].float()[..., None]
        rows = slice(r * tokens, (r + 1) * tokens)
        out[rows] = _softmax_product(s["q"][rows].float(), k, v, s["scale"], n - tokens + 1).half()
    return out


def _plain_prompt(s):
    out = torch.empty(s["q"].shape[0], s["heads"], s["v_dim"], dtype=torch.float16, device=DEVICE)
    for a, b in zip(s["host_cu"], s["host_cu"][1:]):
        out[a:b] = _softmax_product(s["q"][a:b].float(), s["k"][a:b].float(), s["v"][a:b].float(), s["scale"], 1).half()
    return out


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    cached, new = [a for a, _ in _requests(case)], [b for _, b in _requests(case)]
    if kind == "assign":
        held = sum(_pages_of([a for a, b in zip(cached, new) if b < 0], case["page"]))
        need = sum(_pages_of([a + max(b, 0) for a, b in zip(cached, new)], case["page"])) - sum(_pages_of(cached, case["page"]))
        tokens = sum(max(b, 0) for b in new)
        return {"bytes": 12 * tokens + 24 * len(new) + 8 * (held + need), "flops": 0}
    values = case["head_dim"] + case["v_dim"]
    if kind == "store":   # the rows once in and once out, their place, what the cache holds of them
        vectors = sum(new) * case["kv_heads"]
        return {"bytes": vectors * (4 * values + values / 2 + 4) + 8 * sum(new), "flops": 4 * vectors * values}
    pairs = sum(b * a + b * (b + 1) // 2 for a, b in zip(cached, new))
    rows = 2 * case["heads"] * values * sum(new)
    if kind == "attend":
        held = (sum(cached) + sum(new)) * case["kv_heads"] * (values / 2 + 4)
    else:
        held = 2 * case["kv_heads"] * values * sum(new)
    return {"bytes": rows + held, "flops": 2 * pairs * case["heads"] * values}


# ---------------------------------------------------------------------------------------------
# the operators' definitions
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    return {"assign": _exact_assign, "store": _exact_store, "attend": _exact_attend, "prompt": _exact_prompt}[case["kind"]](case, seed)


def _exact_assign(case, seed):
    new, lengths, table, free_pages, count, most = _assign_inputs(case, seed)
    page = case["page"]
    new, lengths, table = new.tolist(), lengths.tolist(), [row for row in table.tolist()]
    stack, memory = free_pages.tolist()[: int(count)], free_pages.tolist()
    after = list(lengths)
    for r, n in enumerate(new):
        if n < 0:
            for page_number in table[r][: -(-lengths[r] // page)]:
                memory[len(stack)] = page_number
                stack.append(page_number)
            after[r] = 0
    slots, positions, refused, cu, asked = [-1] * most, [0] * most, [0] * len(new), [0], 0
    available, used = len(stack), 0
    for r, n in enumerate(new):
        begin = cu[-1]
        end = begin + max(n, 0)
        cu.append(min(end, most) if end <= most else most)
        if n <= 0:
            continue
        have, want = -(-lengths[r] // page), -(-(lengths[r] + n) // page)
        if want > len(table[r]) or lengths[r] + n > len(table[r]) * page or end > most:
            refused[r] = 1
            continue
        asked += want - have
        if want > have and asked > available:
            refused[r] = 1
            continue
        for j in range(have, want):
            table[r][j] = stack.pop()
            used += 1
        for i in range(n):
            position = lengths[r] + i
            positions[begin + i] = position
            slots[begin + i] = table[r][position // page] * page + position % page
        after[r] = lengths[r] + n
    as_int = dict(dtype=torch.int32, device=DEVICE)
    return dict(slots=torch.tensor(slots, dtype=torch.int64, device=DEVICE), positions=torch.tensor(positions, **as_int),
                cu=torch.tensor(cu, **as_int), refused=torch.tensor(refused, **as_int), lengths=torch.tensor(after, **as_int),
                count=torch.tensor([available - used], **as_int), table=torch.tensor(table, **as_int),
                free_pages=torch.tensor(memory, **as_int))


def _as_held(x):
    """the values that the cache holds for the vectors x, in 64 bits"""
    wide = x.to(torch.float64)
    largest = torch.maximum(wide.max(dim=-1).values, -wide.min(dim=-1).values)
    step = (largest / 7.5).to(torch.float16).to(torch.float64).unsqueeze(-1)
    steps = torch.where(step == 0, torch.zeros_like(wide), wide / torch.where(step == 0, torch.ones_like(step), step))
    return step * steps.round().clamp(min=-8.0, max=7.0)


def _exact_store(case, seed):
    k, v = _store_inputs(case, seed)[:2]
    return dict(k=_as_held(k), v=_as_held(v))


def _exact_rows(q, k, v, scale, offset, out):
    """q [t, h, d] of one sequence, 64-bit keys and values, row i sees keys up to offset + i"""
    group = q.shape[1] // k.shape[1]
    for h in range(q.shape[1]):
        keys, values = k[:, h // group], v[:, h // group]
        for at in range(0, q.shape[0], 2048):
            rows = q[at:at + 2048, h].to(torch.float64)
            seen = min(keys.shape[0], offset + at + rows.shape[0])
            weight = rows @ keys[:seen].T * scale
            last = offset + at + torch.arange(rows.shape[0], device=q.device)
            weight = torch.where(torch.arange(seen, device=q.device)[None, :] <= last[:, None], weight, -math.inf)
            weight = torch.softmax(weight, dim=-1)
            out[at:at + 2048, h] = weight @ values[:seen]


def _exact_attend(case, seed):
    q, _, _, lengths, keys_values = _attend_inputs(case, seed)
    tokens = case["tokens"]
    out = torch.empty(q.shape[0], case["heads"], case["v_dim"], dtype=torch.float64, device=DEVICE)
    for r, n in enumerate(lengths):
        k, v = keys_values(r)
        rows = slice(r * tokens, (r + 1) * tokens)
        _exact_rows(q[rows], _as_held(k), _as_held(v), case["head_dim"] ** -0.5, n - tokens, out[rows])
    return out


def _exact_prompt(case, seed):
    q, k, v, cu = _prompt_inputs(case, seed)
    out = torch.empty(q.shape[0], case["heads"], case["v_dim"], dtype=torch.float64, device=DEVICE)
    for a, b in zip(cu, cu[1:]):
        _exact_rows(q[a:b], k[a:b].double(), v[a:b].double(), case["head_dim"] ** -0.5, 0, out[a:b])
    return out
