"""Attention in 64 bits on the CPU, and how far an f32 result may be from it."""
from __future__ import annotations

import math

import torch

U = 2.0 ** -24  # half a step of binary32


def attend(q, k, v, seen, scale=None):
    """q [n, Hq, D], k, v [m, Hk, D], seen [n, m] -> (out, bound), both [n, Hq, D] float64 on the CPU.

    The bound counts roundings, for a kernel that keeps f32 accumulators rounded at most once per 4 products, scores
    and weights in f32 and its binary16 operands in two parts of 22 bits together:
      score error   d <= u * (A * (D/4 + 4 + 4) + |s| + 4), A = scale * sum_i |q_i k_i| (4u = 2^-22 for the parts of q)
      output error  <= (2 d + u * (m/4 + 16)) * sum_j p_j |v_j|, the weights' own parts and exp2's step among the 16.
    """
    n, Hq, D = q.shape
    m, Hk, _ = k.shape
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    seen = seen.cpu()
    out = torch.zeros(n, Hq, D, dtype=torch.float64)
    bound = torch.zeros(n, Hq, D, dtype=torch.float64)
    if m == 0 or n == 0:
        return out, bound
    some = seen.any(1)
    for h in range(Hq):
        g = h // (Hq // Hk)
        # a key that a row does not see takes no part, whatever it holds
        s = torch.where(seen, (q[:, h] @ torch.nan_to_num(k[:, g]).T) * scale, -math.inf)
        A = torch.where(seen, (q[:, h].abs() @ torch.nan_to_num(k[:, g]).abs().T) * abs(scale), 0.0)
        top = torch.where(some, s.amax(1), 0.0)
        p = torch.exp(s - top[:, None])
        den = torch.where(some, p.sum(1), 1.0)
        p = p / den[:, None]
        vz = torch.nan_to_num(v[:, g], nan=0.0, posinf=0.0, neginf=0.0)
        out[:, h] = p @ vz
        d = U * (A * (D / 4 + 8) + torch.where(seen, s.abs(), 0.0) + 4)
        bound[:, h] = (2 * d.amax(1) + U * (m / 4 + 16))[:, None] * (p @ vz.abs()) + 1e-37
    return out, bound


def causal(n, m):
    i, j = torch.arange(n)[:, None], torch.arange(m)[None, :]
    return j <= i + (m - n)


def check(got, want, bound, what=""):
    err = (got.detach().cpu().double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float((err / bound).max()):.2f} "
                           f"bounds, first at {tuple(int(x) for x in bad.nonzero()[0])}")
