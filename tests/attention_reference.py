"""Plain 64-bit implementations of the attention operators, on the CPU, and how far an fp16 kernel may be from them."""
import torch

HALF_STEP = 2.0 ** -11   # fp16: a rounding is off by at most half a step, eps / 2 of the value


def as_held(x):
    """(values, scales) that the 4-bit cache holds for the vectors along the last axis"""
    w = x.double()
    scale = (w.abs().amax(-1) * 2 / 15).half()
    s = scale.double().unsqueeze(-1)
    c = torch.where(s > 0, torch.round(w / s.clamp_min(1e-300)), torch.zeros_like(w)).clamp(-8, 7)
    bad = ~torch.isfinite(w).all(-1)
    scale[bad] = float("nan")
    return torch.where(bad.unsqueeze(-1), torch.full_like(w, float("nan")), c * s), scale


def attention(q, k, v, scale, first_limit):
    """One sequence: q [t, h, d], k [n, g, d], v [n, g, e]; row i sees keys 0 .. first_limit + i - 1.
    Returns (o [t, h, e], a [t, h, e] = sum p |v| / sum p, spread [t, h] = max over keys of sum |q||k| scale)"""
    t, h, d = q.shape
    n, g, e = v.shape
    q, k, v = q.double(), k.double(), v.double()
    o, a, spread = torch.zeros(t, h, e, dtype=torch.float64), torch.zeros(t, h, e, dtype=torch.float64), torch.zeros(t, h, dtype=torch.float64)
    for i in range(t):
        seen = max(0, min(n, first_limit + i))
        if seen == 0:
            continue
        for head in range(h):
            kk, vv = k[:seen, head // (h // g)], v[:seen, head // (h // g)]
            s = kk @ q[i, head] * scale
            p = torch.softmax(s, 0)
            o[i, head] = p @ vv
            a[i, head] = p @ vv.abs()
            spread[i, head] = (kk.abs() @ q[i, head].abs()).max() * scale
    return o, a, spread


def bound(o, a, spread, keys, held=None):
    """The result's rounding (half a step of o); the weights' rounding to fp16 in front of the second product (half a step of each
    term, a = sum p |v|) and, below fp16's normal range, 2^-25 of the largest weight for each key; scores off by their fp32
    sums (at most 2^-23 of sum |q||k| for 128 terms added in blocks, and as much for the scale) change weights by that much,
    numerator and denominator; fp32 sums over the keys, a wave's share of them one after the other.  Held values are summed as
    s c and 8 s apart (`held` = sum p s), each with the fp32 error of such a sum."""
    sums = 2.0 ** -23 * (keys / 32 + 64)
    tol = HALF_STEP * o.abs() + (HALF_STEP + 4 * 2.0 ** -22 * spread.unsqueeze(-1) + sums) * a + 1e-7
    tol = tol + keys * 2.0 ** -24 * a.amax(-1, keepdim=True)
    if held is not None:
        tol = tol + 16 * sums * held
    return tol


def close_bound(o, a, keys, score_error, smallest):
    """How far the kernels' arithmetic may be from 64 bits, without room for another: the result's rounding (half a step); the
    weights' rounding to fp16 in front of the second product, half a step of each term and, where the sum of weights takes the rounded ones, of
    the sum (a = sum p |v|); below fp16's normal range `smallest` for each key, half of 2^-24 over what the largest weight is lifted to;
    scores off by score_error [t, h] (absolute), in numerator and denominator; fp32 sums over the keys, a lane's quarter of them one
    after the other (an error of 2^-24 each) and some 64 steps to join them; the exponentials (2^-22)."""
    sums = 2.0 ** -24 * (keys / 4 + 64) + 2.0 ** -22
    return HALF_STEP * o.abs() + (HALF_STEP + 2 * score_error.unsqueeze(-1) + 2 * sums) * (a + o.abs()) + keys * smallest.unsqueeze(-1)
