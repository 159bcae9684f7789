"""Windowed attention and its gradients in 64 bits -- TEST INFRASTRUCTURE.

From the definition: query row i of M, at position p = (N - M) + i, sees key j iff
j <= p and (j > p - window or j < sinks).  Each result comes with a bound of
what a kernel may be off by that multiplies in the input type and accumulates
in fp32.
"""
from __future__ import annotations

import math

import torch

from .cache import visible


def reference(q, k, v, window: int, sinks: int = 0, do=None, sm_scale=None,
              few_keys: bool = False) -> dict:
    """One batch entry: q, do (Hq, M, D), k, v (Hk, N, D).  Returns out, lse and,
    with do, dq, dk, dv, and under name + "_bound" their bounds.

    half: half a step of the type (relative), f = 2^-24.
    Scores: D products in fp32, the scale, the base-2 exponent and the
    exponential: a weight is off by the factor 1 + w, w = 2 ((D + 4) f S + 4 f (1 +
    S)), S the largest sum of |q||k| sm_scale (the normalizer's share included).
    out: weights rounded for the product, N terms in fp32, one rounding:
      half |out| + (half + 2 w + 2 N f) sum P |v|.
    dv: the same over M G terms:  half |dv| + (half + 2 w + 2 M G f) sum P |do|.
    dP - delta: D products each, delta from the rounded out:
      u = 2 (D + 2) f sum |do||v| + (D + 2) f sum |do||out| + sum |do| out_bound
    (u per pair); with few_keys (no row block's first row sees more than 128 keys)
    delta is the sum of P dP over the row's N keys instead, and with a = 2 (D + 2) f
    sum |do||v|:  u = a + sum_j P a + (2 w + 2 N f) sum_j P |dP|;
    and dS = P (dP - delta), rounded for its products:
      e = P u + |dS| (half + 2 w + 4 f);
    for dk of a bf16 call P may pass between waves in fp16 (half a step: 2^-11 of its
    value, 2^-25 at least):  e + |dS| 2^-11 + |dP - delta| 2^-25 where the pair is
    visible.
    A weight below 2^-126, fp32's least normal number, counts as 0 (exp2 returns no
    subnormals): that leaves 2^-126 |v| out of out, 2^-126 |do| out of dv and 2^-126
    |dP - delta| out of dS.
    dq: half |dq| + s sum_j (e + 2 N f |dS|) |k|;  dk alike over rows."""
    Hq, M, D = q.shape
    Hk, N = k.shape[:2]
    G = Hq // Hk
    scale = 1.0 / math.sqrt(D) if sm_scale is None else sm_scale
    half, f = torch.finfo(q.dtype).eps / 2, 2.0 ** -24
    tiny = torch.finfo(q.dtype).smallest_normal
    q, k, v = q.double(), k.double(), v.double()
    kx, vx = k.repeat_interleave(G, 0), v.repeat_interleave(G, 0)
    see = visible(torch.arange(N - M, N), N, window, sinks)
    s = (q @ kx.transpose(1, 2)) * scale
    S = float(((q.abs() @ kx.abs().transpose(1, 2)) * abs(scale))[:, see].max()) if see.any() else 0.0
    w = 2 * ((D + 4) * f * S + 4 * f * (1 + S))
    s = s.masked_fill(~see, -math.inf)
    lse = torch.logsumexp(s, -1) if N > 0 else torch.full((Hq, M), -math.inf, dtype=torch.float64)
    P = torch.exp(s - torch.where(torch.isinf(lse), 0.0, lse)[..., None])
    out = P @ vx
    res = {"out": out, "lse": lse}
    least = 2.0 ** -126 * see.double().expand(Hq, M, N)
    res["out_bound"] = half * out.abs() + (half + 2 * w + 2 * N * f) * (1 + half) * (P @ vx.abs()) + least @ vx.abs() + tiny
    res["lse_bound"] = w + N * f + 4 * f * (1 + torch.where(torch.isinf(lse), 0.0, lse.abs()))
    if do is None:
        return res
    do = do.double()
    fold = lambda x: x.reshape(Hk, G, N, D).sum(1)
    dP = do @ vx.transpose(1, 2)
    dS = P * (dP - (do * out).sum(-1, keepdim=True))
    res["dv"] = fold(P.transpose(1, 2) @ do)
    res["dq"] = (dS @ kx) * scale
    res["dk"] = fold(dS.transpose(1, 2) @ q) * scale
    u = 2 * (D + 2) * f * (do.abs() @ vx.abs().transpose(1, 2))
    if few_keys:
        u = u + (P * u).sum(-1, keepdim=True) + (2 * w + 2 * N * f) * (P * dP.abs()).sum(-1, keepdim=True)
    else:
        u = u + ((D + 2) * f * (do * out).abs() + do.abs() * res["out_bound"]).sum(-1, keepdim=True)
    gap = (dP - (do * out).sum(-1, keepdim=True)).abs()
    e = P * u + dS.abs() * (half + 2 * w + 4 * f) + least * gap
    res["dv_bound"] = half * res["dv"].abs() + tiny + (half + 2 * w + 2 * M * G * f) * (1 + half) \
        * fold(P.transpose(1, 2) @ do.abs()) + fold(least.transpose(1, 2) @ do.abs())
    res["dq_bound"] = half * res["dq"].abs() + tiny + (1 + half) * abs(scale) \
        * ((e + 2 * N * f * dS.abs()) @ kx.abs())
    if half == 2.0 ** -8:
        e = e + dS.abs() * 2.0 ** -11 + torch.where(see, 2.0 ** -25, 0.0) * gap
    res["dk_bound"] = half * res["dk"].abs() + tiny + (1 + half) * abs(scale) \
        * fold((e + 2 * M * G * f * dS.abs()).transpose(1, 2) @ q.abs())
    return res
