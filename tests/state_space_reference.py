"""Plain 64-bit implementations of what stands between the projections of a state-space layer, on the CPU, and how far the kernels may
be from them."""
import math

import torch

HALF_STEP = 2.0 ** -11   # fp16: a rounding is off by at most half a step, eps / 2 of the value
LEAST = 2.0 ** -25       # and by half of the smallest subnormal number


def offsets(lengths, first=0):
    out = [first]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def silu(u):
    return u / (1 + torch.exp(-u))


def conv(x, weight, bias, state, activation=True):
    """One sequence: x [t, c], weight [c, w], state [w - 1, c].  Returns (y, tolerance, new state).
    The tolerance: the result's rounding; fp32 sums of w + 1 terms (each addition 2^-24 of their absolute sum), through a function
    whose slope is at most 1.1; the exponential (2^-22, and its argument's rounding, 2^-24 |u|), the quotient (2^-22)."""
    t, w = x.shape[0], weight.shape[1]
    line = torch.cat([state.double(), x.double()])
    u = torch.zeros(t, x.shape[1], dtype=torch.float64) + (bias.double() if bias is not None else 0)
    size = u.abs()
    for k in range(w):
        term = line[k:k + t] * weight[:, k].double()
        u, size = u + term, size + term.abs()
    y = silu(u) if activation else u
    tol = HALF_STEP * y.abs() + LEAST + 1.1 * 2.0 ** -24 * (w + 2) * size + (y.abs() * (2.0 ** -21 + 2.0 ** -23 * u.abs()) if activation else 0)
    return y, tol, line[t:]


def time_steps(dt, dt_bias, softplus=True, limit=(0.0, math.inf)):
    u = dt.double() + (dt_bias.double() if dt_bias is not None else 0)
    if softplus:
        u = u.clamp_min(0) + torch.log1p(torch.exp(-u.abs()))
    return u.clamp(*limit)


def scan(x, dt, a, b, c, d, dt_bias, state, softplus=True, limit=(0.0, math.inf)):
    """One sequence: x [t, h, p], dt [t, h], b and c [t, g, n], state [h, p, n].  Returns (y, its tolerance, new state, its tolerance).
    Beside the state S runs the sum of its terms' sizes, A, and of each size times what the exponents that have faded it sum up to, M.
    y: its rounding, the weights' or the state's to fp16 in front of the products (half a step of each term, of which A c is the sum), and
    2^-14 of A c: fp32 sums of at most 400 terms, exponentials whose argument of up to 2^10 is off by 2^-24.
    S: each term is split in two fp16 numbers (2^-22), its time step off by 2^-21, the sums fp32: 128 products a chunk and some four
    roundings for each chunk of 64 (2^-24 each); every exponent is off by 2^-21 of itself, which M counts."""
    t, h, p = x.shape
    share = h // b.shape[1]
    s = time_steps(dt, dt_bias, softplus, limit)
    S = state.double().clone()
    A, M = S.abs(), torch.zeros_like(S)
    y, tol = torch.zeros(t, h, p, dtype=torch.float64), torch.zeros(t, h, p, dtype=torch.float64)
    b, c = b.double().repeat_interleave(share, 1), c.double().repeat_interleave(share, 1)
    for i in range(t):
        log = (s[i] * a.double())[:, None, None]
        new = (s[i][:, None] * x[i].double())[:, :, None] * b[i][:, None, :]
        M = torch.exp(log) * (M + log.abs() * A)
        S, A = torch.exp(log) * S + new, torch.exp(log) * A + new.abs()
        through = torch.zeros(h, p, dtype=torch.float64) if d is None else d.double()[:, None] * x[i].double()
        y[i] = (S * c[i][:, None, :]).sum(-1) + through
        size = (A * c[i].abs()[:, None, :]).sum(-1)
        tol[i] = HALF_STEP * y[i].abs() + LEAST + (HALF_STEP + 2.0 ** -14) * size + 2.0 ** -22 * through.abs() \
            + 2.0 ** -21 * (M * c[i].abs()[:, None, :]).sum(-1)
    return y, tol, S, A * (2.0 ** -24 * (128 + 4 * (t / 64 + 1)) + 2.0 ** -20) + 2.0 ** -20 * M + 1e-30


def gated_norm(x, z, weight, groups, eps):
    """Returns (y, tolerance): the result's rounding; the gate (2^-21, and 2^-23 |z| by its exponent), in the value itself and, largest of
    the group, in the mean; the sum (a lane's share one after the other, some 40 to join them, 2^-24 each), the root and three products."""
    u = x.double() * silu(z.double())
    grouped = u.view(u.shape[0], groups, -1)
    width = grouped.shape[2]
    y = (grouped / torch.sqrt(grouped.square().mean(-1, keepdim=True) + eps)).view_as(u) * weight.double()
    gate = 2.0 ** -21 + 2.0 ** -23 * z.double().abs()
    most = gate.view_as(grouped).amax(-1, keepdim=True).expand_as(grouped).reshape_as(u)
    return y, HALF_STEP * y.abs() + LEAST + y.abs() * (gate + most + 2.0 ** -24 * (width / 64 + 40) + 2.0 ** -21)
