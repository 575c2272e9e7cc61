"""The C entry points of the cache and of attention refuse what they cannot do before anything is launched (no GPU needed)."""
import ctypes

import pytest

from uniql_amd import _capi


class Cache(ctypes.Structure):
    _fields_ = [("k_codes", ctypes.c_void_p), ("k_scales", ctypes.c_void_p), ("v_codes", ctypes.c_void_p), ("v_scales", ctypes.c_void_p),
                ("pages", ctypes.c_int), ("page_size", ctypes.c_int), ("heads", ctypes.c_int), ("k_dim", ctypes.c_int),
                ("v_dim", ctypes.c_int)]


FAKE = 0x10000


@pytest.fixture(scope="module")
def lib():
    return _capi.load()


def cache(**kw):
    return Cache(**{**dict(k_codes=FAKE, k_scales=FAKE, v_codes=FAKE, v_scales=FAKE, pages=4, page_size=16, heads=2, k_dim=64, v_dim=64), **kw})


BAD_CACHES = [(dict(page_size=24), -2), (dict(page_size=8), -2), (dict(page_size=512), -2), (dict(pages=0), -2), (dict(heads=0), -2),
              (dict(heads=5000), -2), (dict(k_dim=0), -2), (dict(v_dim=-1), -2), (dict(k_dim=129), -5), (dict(v_dim=256), -5)]
BAD_POINTERS = [(dict(k_codes=None), -1), (dict(v_scales=None), -1), (dict(k_codes=FAKE + 4), -3), (dict(k_scales=FAKE + 8), -3)]


def test_assign(lib):
    args = dict(new=FAKE, lengths=FAKE, table=FAKE, free=FAKE, count=FAKE, lengths_out=FAKE, count_out=FAKE, slots=FAKE, positions=FAKE,
                cu=FAKE, refused=FAKE, rows=2, columns=3, pool=4, page=16, most=5, stream=None)

    def call(**kw):
        return lib.uniql_kv_assign_pages(*{**args, **kw}.values())

    for kw, code in [(dict(rows=-1), -2), (dict(columns=0), -2), (dict(columns=(1 << 20) + 1), -2), (dict(pool=-1), -2), (dict(page=15), -2),
                     (dict(most=-1), -2), (dict(most=(1 << 24) + 1), -2), (dict(columns=1 << 20, rows=4096), -2),
                     (dict(columns=1 << 20, rows=1, page=256, new=None), -1)]:
        assert call(**kw) == code, kw
    for name in ("new", "lengths", "table", "free", "count", "lengths_out", "count_out", "slots", "positions", "cu", "refused"):
        assert call(**{name: None}) == -1, name


@pytest.mark.parametrize("kw,code", BAD_CACHES + BAD_POINTERS)
def test_caches(lib, kw, code):
    c = cache(**kw)
    p = ctypes.byref(c)
    store = lambda **a: lib.uniql_kv4_store(*{**dict(k=FAKE, kr=64, kh=64, v=FAKE, vr=64, vh=64, slots=FAKE, cache=p, tokens=1, stream=None), **a}.values())
    load = lambda **a: lib.uniql_kv4_load(*{**dict(cache=p, table=FAKE, cu=FAKE, starts=None, k=FAKE, kr=1, kh=1, v=FAKE, vr=1, vh=1, requests=1,
                                                   columns=1, rows=1, stream=None), **a}.values())
    attend = lambda **a: lib.uniql_kv4_attention(*{**dict(q=FAKE, qr=1, qh=1, cache=p, table=FAKE, lengths=FAKE, cu=FAKE, out=FAKE, outr=1,
                                                          outh=1, accum=FAKE, accum_bytes=1 << 40, temp=FAKE, temp_bytes=1 << 40, rows=1,
                                                          requests=1, columns=1, heads=4, scale=1.0, stream=None), **a}.values())
    if "heads" in kw and kw["heads"] == 5000:
        assert store() == code and load() == code
    else:
        assert store() == code and load() == code and attend() == code
    acc, tmp = ctypes.c_size_t(0), ctypes.c_size_t(0)
    if (kw, code) in BAD_CACHES:
        assert lib.uniql_kv4_attention_workspace(p, 1, 1, 1, 4, ctypes.byref(acc), ctypes.byref(tmp)) == code


def test_store_load_and_attention(lib):
    c = cache()
    p = ctypes.byref(c)
    sizes = dict(k=FAKE, kr=64, kh=64, v=FAKE, vr=64, vh=64, slots=FAKE, cache=p, tokens=1, stream=None)
    store = lambda **a: lib.uniql_kv4_store(*{**sizes, **a}.values())
    assert store(tokens=-1) == -2 and store(k=None) == -1 and store(v=None) == -1 and store(slots=None) == -1 and store(cache=None) == -1
    assert store(tokens=0, k=None) == 0
    load = lambda **a: lib.uniql_kv4_load(*{**dict(cache=p, table=FAKE, cu=FAKE, starts=None, k=FAKE, kr=1, kh=1, v=FAKE, vr=1, vh=1, requests=1,
                                                   columns=1, rows=1, stream=None), **a}.values())
    assert load(rows=-1) == -2 and load(requests=-1) == -2 and load(columns=0) == -2 and load(columns=1 << 20, requests=1 << 12) == -2
    assert load(table=None) == -1 and load(cu=None) == -1 and load(k=None) == -1 and load(v=None) == -1 and load(rows=0, k=None) == 0
    base = dict(q=FAKE, qr=1, qh=1, cache=p, table=FAKE, lengths=FAKE, cu=FAKE, out=FAKE, outr=1, outh=1, accum=FAKE, accum_bytes=1 << 40,
                temp=FAKE, temp_bytes=1 << 40, rows=1, requests=1, columns=1, heads=4, scale=1.0, stream=None)
    attend = lambda **a: lib.uniql_kv4_attention(*{**base, **a}.values())
    assert attend(heads=3) == -2 and attend(heads=0) == -2 and attend(heads=8192) == -2 and attend(rows=-1) == -2 and attend(requests=-1) == -2
    assert attend(cu=None, rows=2) == -2 and attend(columns=0) == -2 and attend(rows=0, q=None) == 0 and attend(requests=0, q=None) == 0
    assert attend(q=None) == -1 and attend(table=None) == -1 and attend(lengths=None) == -1 and attend(out=None) == -1
    acc, tmp = ctypes.c_size_t(0), ctypes.c_size_t(0)
    assert lib.uniql_kv4_attention_workspace(p, 1, 1, 1, 4, None, ctypes.byref(tmp)) == -1
    assert lib.uniql_kv4_attention_workspace(p, 300, 100, 500, 4, ctypes.byref(acc), ctypes.byref(tmp)) == 0
    if tmp.value:
        assert attend(rows=300, requests=100, columns=500, temp_bytes=tmp.value - 1) == -4
        assert attend(rows=300, requests=100, columns=500, accum_bytes=acc.value - 1) == -4
        assert attend(rows=300, requests=100, columns=500, temp=None) == -1


def test_prompt_attention(lib):
    base = dict(q=FAKE, qr=1, qh=1, k=FAKE, kr=1, kh=1, v=FAKE, vr=1, vh=1, cu_q=FAKE, cu_k=FAKE, out=FAKE, outr=1, outh=1, rows=4, k_rows=4,
                sequences=1, heads=4, kv=2, kd=64, vd=64, causal=1, scale=1.0, stream=None)
    call = lambda **a: lib.uniql_prompt_attention(*{**base, **a}.values())
    for name in ("q", "k", "v", "cu_q", "cu_k", "out"):
        assert call(**{name: None}) == -1
    assert call(rows=-1) == -2 and call(k_rows=-1) == -2 and call(sequences=-1) == -2 and call(heads=3) == -2 and call(kv=0) == -2
    assert call(kd=0) == -2 and call(vd=0) == -2 and call(kd=129) == -5 and call(vd=160) == -5 and call(heads=8192) == -2
    assert call(rows=0, q=None) == 0 and call(sequences=0, q=None) == 0


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf"), 1.9e19, -1.9e19, 3e38])
def test_scales_with_which_finite_inputs_have_no_finite_scores(lib, scale):
    """2^64 = 1.845e19: times 128 products of fp16 numbers (2^39) and what the kernels fold in (2^25 and less) it stays below 2^128"""
    p = ctypes.byref(cache())
    args = [FAKE, 1, 1, p, FAKE, FAKE, FAKE, FAKE, 1, 1, FAKE, 1 << 40, FAKE, 1 << 40, 1, 1, 1, 4]
    assert lib.uniql_kv4_attention(*args, scale, None) == -5
    prompt = [FAKE, 1, 1, FAKE, 1, 1, FAKE, 1, 1, FAKE, FAKE, FAKE, 1, 1, 4, 4, 1, 4, 2, 64, 64, 1]
    assert lib.uniql_prompt_attention(*prompt, scale, None) == -5
    # no rows: what is left of the checks passes with the largest scales
    args[14], prompt[14] = 0, 0
    for most in (2.0 ** 64, -2.0 ** 64, 1.0):
        assert lib.uniql_kv4_attention(*args, most, None) == 0 and lib.uniql_prompt_attention(*prompt, most, None) == 0


@pytest.mark.parametrize("count", [(1 << 30) + 1, (1 << 31) - 64, (1 << 31) - 1])
def test_more_requests_than_sums_of_their_numbers_allow(lib, count):
    p = ctypes.byref(cache())
    assert lib.uniql_kv_assign_pages(*[FAKE] * 11, count, 1, 4, 16, 5, None) == -2
    assert lib.uniql_kv4_load(p, FAKE, FAKE, None, FAKE, 1, 1, FAKE, 1, 1, count, 1, 1, None) == -2
    acc, tmp = ctypes.c_size_t(0), ctypes.c_size_t(0)
    assert lib.uniql_kv4_attention_workspace(p, 1, count, 1, 4, ctypes.byref(acc), ctypes.byref(tmp)) == -2
    assert lib.uniql_kv4_attention(FAKE, 1, 1, p, FAKE, FAKE, FAKE, FAKE, 1, 1, FAKE, 1 << 40, FAKE, 1 << 40, 1, count, 1, 4, 1.0, None) == -2
    assert lib.uniql_prompt_attention(FAKE, 1, 1, FAKE, 1, 1, FAKE, 1, 1, FAKE, FAKE, FAKE, 1, 1, 4, 4, count, 4, 2, 64, 64, 1, 1.0, None) == -2


@pytest.mark.parametrize("heads,q_heads", [(1, 4), (8, 32), (32, 32), (600, 600)])
def test_scratch_does_not_grow_with_the_rows(lib, heads, q_heads):
    """only rows that several workgroups share need some, and those are at most two for each of the 512 workgroups that a call is shared
    out to (rounded up to whole ones a head): 8320 bytes and a word each"""
    p = ctypes.byref(cache(heads=heads))
    most = 2 * -(-512 // heads) * heads
    for rows, requests in ((1, 1), (64, 64), (500, 500), (500, 3), (16384, 1), (16384, 300), (131072, 5)):
        acc, tmp = ctypes.c_size_t(0), ctypes.c_size_t(0)
        assert lib.uniql_kv4_attention_workspace(p, rows, requests, 64, q_heads, ctypes.byref(acc), ctypes.byref(tmp)) == 0
        assert 0 < tmp.value <= most * 8320 and 0 < acc.value <= 4 * most + 7
        if rows == 1:
            assert tmp.value < most * 8320 or heads >= 512


def test_heads_without_width_are_refused_as_anything_else(lib):
    """also where the scale is left to the width"""
    import torch
    from uniql_amd import ops
    x = torch.zeros(3, 2, 0, dtype=torch.float16)
    i = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: ops.prompt_attention(x, x, x, i), lambda: ops.kv4_attention(x, i, x, i, x, i, i, 64),
                 lambda: ops.prompt_attention(x[0, 0, 0:].sum(), x, x, i)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
