"""Scores so large that neighbouring fp32 numbers are further apart than the room that the weights have: finite queries and keys
give finite results, and where one key's score is beyond all others by more than any weight can show, that key's values."""
import pytest
import torch

from tests.attention_reference import as_held, attention, bound

pytestmark = pytest.mark.gpu
SIZES = [2.0 ** e for e in (18, 21, 22, 23, 24, 25, 26, 27, 28, 29, 31, 36)]


def ordered(values, order, seed=0):
    if order == "falling":
        return values.flip(0)
    return values if order == "rising" else values[torch.randperm(len(values), generator=torch.Generator().manual_seed(seed))]


def strongest(size, turned):
    """the first key of the largest (turned: smallest) size among those up to each"""
    return torch.tensor([int((size[:i + 1].argmin if turned else size[:i + 1].argmax)()) for i in range(len(size))])


@pytest.mark.parametrize("score", SIZES)
@pytest.mark.parametrize("turned", [False, True])
def test_prompts(gpu, score, turned):
    """Keys of one number each, 8 apart: the scores of two keys differ by a 256th of the largest and more, thousands; their fp32
    errors are 2^-20 of it.  A weight of 1 and zeros: sum and quotient give the values themselves."""
    from uniql_amd.attention import prompt_attention
    n = 200
    gen = torch.Generator().manual_seed(1)
    cu = torch.tensor([0, n], dtype=torch.int32, device=gpu)
    for order in ("rising", "falling", "mixed"):
        size = ordered(1000.0 + 8 * torch.arange(n), order)
        k = size.view(n, 1, 1).expand(n, 1, 64).half().contiguous()
        v = torch.randn(n, 1, 48, generator=gen).half()
        q = ((-1.0 if turned else 1.0) * (1 + torch.arange(n) / 256).view(n, 1, 1)).expand(n, 2, 64).half().contiguous()
        got = prompt_attention(q.to(gpu), k.to(gpu), v.to(gpu), cu, scale=1.1 * score / 2 ** 17).cpu()
        want = v[strongest(size, turned)].expand(n, 2, 48)
        assert torch.equal(got, want), (order, int((got != want).any(-1).any(-1).sum()))


@pytest.mark.parametrize("score", SIZES)
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("n,requests", [(50, 2), (700, 1), (700, 600)])
def test_over_the_cache(gpu, score, turned, n, requests):
    """As above, with values from 1e-3 to 1e3.  Rounding: of the one weight times its scale and of the result, half a step each."""
    from uniql_amd.quantize.quant_kv_cache import W4KVCache
    gen = torch.Generator().manual_seed(2)
    pages = -(-n // 16)
    table = torch.randperm(pages, generator=gen).to(torch.int32).expand(requests, pages).contiguous()
    slots = table[0].long()[torch.arange(n) // 16] * 16 + torch.arange(n) % 16
    lengths = torch.full((requests,), n, dtype=torch.int32, device=gpu)
    for order in ("rising", "falling", "mixed"):
        size = ordered(1000.0 + 8 * torch.arange(n), order)
        k = size.view(n, 1, 1).expand(n, 1, 64).half().contiguous()
        v = (torch.randn(n, 1, 40, generator=gen) * 10 ** (6 * torch.rand(n, 1, 1, generator=gen) - 3)).half()
        cache = W4KVCache(pages, 16, 1, 64, 40, device=gpu)
        cache.store(k.to(gpu), v.to(gpu), slots.to(gpu))
        q = torch.full((requests, 2, 64), -1.0 if turned else 1.0, device=gpu).half()
        got = cache.attend(q, table.to(gpu), lengths, scale=1.1 * score / 2 ** 17).cpu().double()
        held_k, held_v = as_held(k)[0], as_held(v)[0]
        want = held_v[int((held_k[:, 0, 0].argmin if turned else held_k[:, 0, 0].argmax)()), 0]
        assert ((got - want).abs() <= 2 ** -10 * want.abs() + 2 ** -25).all(), (order, float((got - want).abs().max()))


NEAR = [0, 3, 70, 130, 199]


def near_and_far(far):
    """keys along a direction that all queries share, far behind the few that stand on their own"""
    gen = torch.Generator().manual_seed(4)
    k = torch.zeros(200, 1, 64)
    k[:, :, 0] = -far * (1 + torch.arange(200).flip(0).view(-1, 1) / 200)
    k[NEAR] = torch.cat((torch.zeros(len(NEAR), 1, 1), torch.randn(len(NEAR), 1, 63, generator=gen)), 2)
    q = torch.cat((torch.full((200, 2, 1), 30000.0), torch.randn(200, 2, 63, generator=gen)), 2)
    return q.half(), k.half(), torch.randn(200, 1, 48, generator=gen).half()


@pytest.mark.parametrize("far", [100.0, 3000.0, 30000.0])
@pytest.mark.parametrize("causal", [True, False])
def test_prompts_with_scores_far_below(gpu, far, causal):
    """most scores are 10^6 to 10^9 below those of five keys, which alone have weight; the tolerance is that of attention over them"""
    from uniql_amd.attention import prompt_attention
    q, k, v = near_and_far(far)
    cu = torch.tensor([0, 200], dtype=torch.int32, device=gpu)
    for first in (0, 1):                  # the five in front of or behind the others, too
        keys = torch.arange(200) if first == 0 else torch.arange(200).flip(0)
        got = prompt_attention(q.to(gpu), k[keys].to(gpu), v[keys].to(gpu), cu, causal=causal, scale=0.3).cpu().double()
        near = [int((keys == j).nonzero()) for j in NEAR]
        for i in range(200):
            seen = sorted(j for j in near if j <= i or not causal)
            if not seen:
                continue
            o, mean_abs, spread = attention(q[i:i + 1, :, 1:], k[keys][seen, :, 1:], v[keys][seen], 0.3, len(seen))
            assert ((got[i] - o[0]).abs() <= bound(o, mean_abs, spread, 200)[0]).all(), (first, i)


def test_near_rows_beside_far_ones(gpu):
    """a block of rows some of which have far scores, and infinities behind the causal border: the others' results are what they are"""
    from uniql_amd.attention import prompt_attention
    gen = torch.Generator().manual_seed(6)
    q, k, v = (torch.randn(150, 2, 64, generator=gen).half() for _ in range(3))
    v[140:] = float("inf")
    far = q.clone()
    far[::5] *= 20000
    k[:, :, 0] = 2000.0 + torch.arange(150).view(-1, 1)
    q[:, :, 0], far[:, :, 0] = 0, 0
    far[::5, :, 0] = 30000.0
    cu = torch.tensor([0, 150], dtype=torch.int32, device=gpu)
    got = prompt_attention(far.to(gpu), k.to(gpu), v.to(gpu), cu, scale=0.2).cpu()
    o, mean_abs, spread = attention(q, k, v, 0.2, 1)
    rows = torch.tensor([i for i in range(140) if i % 5])
    k[:, :, 0] = 0
    tol = bound(*attention(q, k, v, 0.2, 1), 150)
    assert ((got.double() - o).abs() <= tol)[rows].all()
    k[:, :, 0] = 2000.0 + torch.arange(150).view(-1, 1)
    for i in range(0, 140, 5):     # scores of 10^7, some fp32 roundings of 1 each away: a key that is ahead by 200 has all the weight
        for h in range(2):
            s, at = torch.sort(k[:i + 1, h].double() @ far[i, h].double() * 0.2, descending=True)
            if not far[i, h].isfinite().all():
                assert got[i, h].isnan().all()
            elif i == 0 or s[0] - s[1] > 200:
                assert torch.equal(got[i, h], v[at[0], h])


@pytest.mark.parametrize("scale", [2.0 ** 64, -2.0 ** 64])
@pytest.mark.parametrize("largest", [3.0, 65504.0])
def test_the_largest_scale(gpu, scale, largest):
    """finite scores of up to 2^104, each further from the next than any weight reaches"""
    from uniql_amd.attention import prompt_attention
    from uniql_amd.quantize.quant_kv_cache import W4KVCache
    gen = torch.Generator().manual_seed(3)
    size = ordered(largest * (1 + torch.arange(100)) / 100, "mixed")
    k = size.view(100, 1, 1).expand(100, 1, 128).half().contiguous()
    v = torch.randn(100, 1, 40, generator=gen).half()
    q = torch.full((1, 2, 128), largest).half().to(gpu)
    at = int(k[:, 0, 0].argmax() if scale > 0 else k[:, 0, 0].argmin())
    cu = [torch.tensor([0, n], dtype=torch.int32, device=gpu) for n in (1, 100)]
    for causal in (True, False):
        got = prompt_attention(q, k.to(gpu), v.to(gpu), *cu, causal=causal, scale=scale).cpu()
        assert torch.equal(got, v[at].expand(1, 2, 40))
    cache = W4KVCache(7, 16, 1, 128, 40, device=gpu)
    cache.store(k.to(gpu), v.to(gpu), torch.arange(100, device=gpu))
    got = cache.attend(q, torch.arange(7, dtype=torch.int32, device=gpu)[None], cu[1][1:], scale=scale).cpu().double()
    want = as_held(v)[0][at, 0]
    assert ((got - want).abs() <= 2 ** -10 * want.abs() + 2 ** -25).all()
