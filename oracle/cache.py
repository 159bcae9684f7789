"""The quantised KV cache and windowed attention in 64 bits -- TEST INFRASTRUCTURE.

Written from the definitions (include/fas.h), on the CPU, independently of the
package: codes as a sorted list of values, rounding by distance, attention by
masked softmax.
"""
from __future__ import annotations

import math

import torch

BLOCK = 32
TOP = {4: 6.0, 8: 448.0}
EXP_MIN = -126
EXP_MAX = {(torch.float16, 4): 13, (torch.float16, 8): 7, (torch.bfloat16, 4): 125,
           (torch.bfloat16, 8): 119}


def magnitudes(bits: int) -> torch.Tensor:
    """Values of the codes without their sign bit, ascending (8 bits: without NaN)."""
    if bits == 4:
        return torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    return torch.tensor([m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
                         for e in range(16) for m in range(8)][:-1], dtype=torch.float64)


def blocks(x: torch.Tensor) -> torch.Tensor:
    D = x.shape[-1]
    return x.reshape(*x.shape[:-1], max(1, D // BLOCK), min(D, BLOCK))


def quantise(x: torch.Tensor, bits: int):
    """(codes, scales) of rows x (..., D), as the cache's bytes."""
    y = blocks(x.double())
    bad = ~torch.isfinite(y).all(-1)
    y = torch.where(bad[..., None], 0.0, y)
    amax = y.abs().amax(-1)
    exp = torch.full(amax.shape, EXP_MIN, dtype=torch.int64)
    for e in range(EXP_MIN, EXP_MAX[x.dtype, bits]):  # the least that does not clip
        exp = torch.where(amax > TOP[bits] * 2.0 ** e, e + 1, exp)
    a = y.abs() / torch.exp2(exp.double())[..., None]
    grid = magnitudes(bits)
    up = torch.searchsorted(grid, a.contiguous()).clamp(max=len(grid) - 1)
    down = (up - 1).clamp(min=0)
    dist_up, dist_down = (grid[up] - a).abs(), (a - grid[down]).abs()
    tie = torch.where(up % 2 == 0, up, down)
    code = torch.where(dist_up < dist_down, up, torch.where(dist_down < dist_up, down, tie))
    code = (code + torch.where(torch.signbit(y), 1 << (bits - 1), 0)).reshape(x.shape)
    code = torch.where(bad[..., None].expand(y.shape).reshape(x.shape), 0, code).to(torch.uint8)
    if bits == 4:
        code = code[..., 0::2] + 16 * code[..., 1::2]
    return code, torch.where(bad, 255, exp + 127).to(torch.uint8)


def decode(codes: torch.Tensor, scales: torch.Tensor, bits: int) -> torch.Tensor:
    """Values of cache bytes, in 64 bits."""
    if bits == 4:
        codes = torch.stack((codes % 16, codes // 16), -1).flatten(-2)
    sign = 1 << (bits - 1)
    mag = magnitudes(bits)
    if bits == 8:
        mag = torch.cat((mag, torch.tensor([math.nan], dtype=torch.float64)))
    val = mag[(codes % sign).long()] * torch.where(codes >= sign, -1.0, 1.0)
    s = torch.exp2(scales.double() - 127)
    s = torch.where(scales == 255, math.nan, s)
    return (blocks(val) * s[..., None]).flatten(-2)


def visible(pos: torch.Tensor, N: int, window: int, sinks: int) -> torch.Tensor:
    """(rows, N): position pos sees key j iff j <= pos and, with a window,
    (j > pos - window or j < sinks)."""
    j = torch.arange(N)
    ok = j[None] <= pos[:, None]
    return ok if not window else ok & ((j[None] > pos[:, None] - window) | (j[None] < sinks))


def attend(q, k, v, pos, window: int = 0, sinks: int = 0, sm_scale=None):
    """One sequence: q (Hq, M, D), k and v (Hk, N, D), pos (M,); rows at a negative
    position see nothing.  Keys that a row does not see do not enter its result,
    whatever they hold.  Returns a dict: out, lse, and what the error bounds
    need: absv (the weights' sum over |v|) and score (the largest sum of |q||k|
    sm_scale of a visible pair)."""
    Hq, M, D = q.shape
    Hk, N = k.shape[:2]
    G = Hq // Hk
    scale = 1.0 / math.sqrt(D) if sm_scale is None else sm_scale
    q, k, v = q.double(), k.double(), v.double()
    out, absv = torch.zeros(Hq, M, D, dtype=torch.float64), torch.zeros(Hq, M, D, dtype=torch.float64)
    lse = torch.full((Hq, M), -math.inf, dtype=torch.float64)
    score = 0.0
    see = visible(pos, N, window, sinks)
    for h in range(Hq):
        for i in range(M):
            idx = see[i].nonzero()[:, 0]
            if len(idx) == 0:
                continue
            ks, vs = k[h // G, idx], v[h // G, idx]
            s = (ks @ q[h, i]) * scale
            lse[h, i] = torch.logsumexp(s, 0)
            w = torch.softmax(s, 0)
            out[h, i], absv[h, i] = w @ vs, w @ vs.abs()
            score = max(score, float((ks.abs() @ q[h, i].abs()).max()) * abs(scale))
    return {"out": out, "lse": lse, "absv": absv, "score": score}


def attend_bounds(ref: dict, dtype: torch.dtype, D: int, N: int):
    """(bound of out's error, bound of lse's), elementwise, by arithmetic.

    A score is a sum of D products accumulated in fp32, once more rounded by the
    scale and by the base-2 exponent: |ds| <= (D + 4) 2^-24 * score, and with the
    exponential's own rounding a weight is off by the factor 1 + d, d = 2 (|ds| +
    2^-22 (1 + score)).  The weights are rounded to the type for the product (half
    a step), their products and their sum are accumulated in fp32 over N keys,
    and the result is rounded to the type:
      |do| <= half * |out| + (half + 2 d + 2 N 2^-24) * absv;
      |dlse| <= d + N 2^-24 + 2^-22 (1 + |lse|)."""
    half = torch.finfo(dtype).eps / 2
    d = 2 * ((D + 4) * 2.0 ** -24 * ref["score"] + 2.0 ** -22 * (1 + ref["score"]))
    tiny = torch.finfo(dtype).smallest_normal  # results below it round in absolute steps
    out = half * ref["out"].abs() + (half + 2 * d + 2 * N * 2.0 ** -24) * ref["absv"] * (1 + half) + tiny
    lse = d + N * 2.0 ** -24 + 2.0 ** -22 * (1 + torch.where(torch.isinf(ref["lse"]), 0.0, ref["lse"].abs()))
    return out, lse
