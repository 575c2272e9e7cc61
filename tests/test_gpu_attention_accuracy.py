"""Attention against 64 bits with bounds that leave no room for coarser arithmetic than the kernels' own."""
import pytest
import torch

from tests.attention_reference import HALF_STEP, as_held, attention, close_bound
from tests.test_gpu_kv_attention import Problem
from tests.test_gpu_prompt_attention import problem, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths,h,g,d,e,page", [
    ([4100, 33], 4, 1, 128, 128, 64), ([9000], 8, 8, 64, 64, 256), ([300] * 70, 4, 2, 108, 100, 16), ([1500, 700, 2], 6, 3, 33, 126, 32),
])
@pytest.mark.parametrize("sharp", [0.0, 0.5, 3.0])
def test_over_the_cache(gpu, lengths, h, g, d, e, page, sharp):
    """Scores: sums of d products of q and codes up to 15, and of 8 q, each rounded to fp32 (at most d steps of 2^-24 of the sum of
    the magnitudes, 23 sum|q| s), then four roundings.  Weights: the largest one times its scale is lifted to 2^5 and more; codes are
    8 at most."""
    p = Problem(gpu, lengths, [1] * len(lengths), h, g, d, e, page, seed=h, sharp=sharp)
    got, scale = p.run().cpu().double(), d ** -0.5
    for r, n in enumerate(lengths[:5]):
        k, k_scales = as_held(p.k[r])
        v, v_scales = as_held(p.v[r])
        q = p.q[r:r + 1]
        o, a, _ = attention(q, k, v, scale, n)
        score_error, smallest = torch.zeros(1, h, dtype=torch.float64), torch.zeros(1, h, dtype=torch.float64)
        for head in range(h):
            kv = head // (h // g)
            weight = torch.softmax(k[:, kv] @ q[0, head].double() * scale, 0)
            reach = 23 * float(k_scales[:, kv].double().max()) * float(q[0, head].double().abs().sum()) * scale
            score_error[0, head] = 2.0 ** -24 * (d / 8 + 8) * reach
            smallest[0, head] = 2.0 ** -25 * 8 * 2.0 ** -5 * float((weight * v_scales[:, kv].double()).max())
        assert ((got[r] - o[0]).abs() <= close_bound(o, a, n, score_error, smallest)[0]).all(), (r, n)


@pytest.mark.parametrize("length,h,g,d,e", [(700, 2, 1, 128, 128), (333, 4, 4, 108, 108), (1500, 1, 1, 64, 64), (513, 3, 1, 33, 100)])
@pytest.mark.parametrize("sharp", [0.0, 0.5, 3.0])
def test_prompts(gpu, length, h, g, d, e, sharp):
    """Scores: fp32 sums of exact products; the largest weight is lifted to 2^6 and more."""
    q, k, v, cu, _ = problem([length], [length], h, g, d, e, seed=d, sharp=sharp)
    got = run(gpu, q, k, v, cu, None).cpu().double()
    o, a, spread = attention(q, k, v, d ** -0.5, 1)
    smallest = torch.full((length, h), 2.0 ** -25 * 2.0 ** -6 * float(v.double().abs().max()), dtype=torch.float64)
    tol = close_bound(o, a, length, 2.0 ** -24 * (d / 8 + 8) * spread, smallest)
    assert ((got - o).abs() <= tol).all(), float(((got - o).abs() - tol).max())


def test_many_small_weights_beside_a_large_one_in_a_wave(gpu):
    """512 requests over the same million positions, so that each of a workgroup's four waves goes through a quarter of them: it finds one
    position of weight 1 and value -1 first, then a quarter million of 2^-25.5 and 1, which without the lift by 2^6 round to nothing (their
    product with the values' scale is 2^-26.4 then) and count 0.011 together.  Rounding: the large weights' and the result's half step; of the
    small ones, which are 12 steps of 2^-24, half a step of those; in the lane that has the large weight an fp32 sum that the small ones, a
    sixteenth of all, are too small for; 8192 fp32 sums of products a wave, half a step each."""
    from uniql_amd.quantize.quant_kv_cache import W4KVCache
    n, requests = 1 << 20, 512
    k, v = torch.zeros(n, 1, 32).half(), torch.ones(n, 1, 32).half()
    large = torch.tensor([10, 74, 138, 202])
    k[large], v[large] = 1.0, -1.0
    cache = W4KVCache(n // 256, 256, 1, 32, 32, device=gpu)
    cache.store(k.to(gpu), v.to(gpu), torch.arange(n, device=gpu))
    held_k, held_v = as_held(k[:12])[0][10, 0], as_held(v[:12])[0][:, 0, 0]
    scale = 25.5 * 0.6931471805599453 / float(held_k.sum())
    table = torch.arange(n // 256, dtype=torch.int32, device=gpu).expand(requests, -1).contiguous()
    got = cache.attend(torch.ones(requests, 2, 32, device=gpu).half(), table, torch.full((requests,), n, dtype=torch.int32, device=gpu),
                       scale=scale).cpu().double()
    small = (n - 4) * 2.0 ** -25.5
    want = float((4 * held_v[10] + small * held_v[0]) / (4 + small))
    lost = small / (4 + small) * float(held_v[0] - held_v[10])
    tol = (2 * HALF_STEP + n / 16 * 2.0 ** -25.5 + 8192 * 2.0 ** -24) * abs(want) + lost / 24
    assert lost > 2 * tol
    assert ((got - want).abs() <= tol).all(), (float(want), float((got - want).abs().max()), tol)
