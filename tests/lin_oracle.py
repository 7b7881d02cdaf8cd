"""Linear attention with a decay per head in 64 bits, token by token, with the
sums of absolute values that the tests' tolerances are made of."""
from __future__ import annotations

import torch


def steps(q, k, v, g, S, scale):
    """q, k [T, Hqk, dk], v [T, Hv, dv], g [T, Hv] log gates, S [Hv, dk, dv].

    Returns (o, S, o_abs, S_abs) in float64: o_abs and S_abs are the same sums
    of the terms' absolute values."""
    T, Hv, dv = v.shape
    group = Hv // q.shape[1]
    q, k = (x.double().repeat_interleave(group, 1) for x in (q, k))
    v, S = v.double(), S.double().clone()
    A = S.abs()
    a = g.double().exp()
    o, oa = torch.zeros(T, Hv, dv, dtype=torch.float64), torch.zeros(T, Hv, dv, dtype=torch.float64)
    for t in range(T):
        S = a[t][:, None, None] * S + k[t][:, :, None] * v[t][:, None, :]
        A = a[t][:, None, None] * A + (k[t][:, :, None] * v[t][:, None, :]).abs()
        o[t] = scale * (q[t][:, :, None] * S).sum(1)
        oa[t] = abs(scale) * (q[t][:, :, None].abs() * A).sum(1)
    return o, S, oa, A


def half_step(dtype):
    """The largest relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2
