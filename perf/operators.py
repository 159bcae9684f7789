"""Performance cases of the windowed attention and the quantised KV cache.

`listed` names the cases, `draw` gives more of the same ranges, `prepare` makes
what a user's program has in hand before the call, `run` makes one pass,
`work` says what a pass cannot do without and `exact` gives its outputs from
the definition in 64 bits.  With `own` false `run` computes the operators in
their plain form (elementary torch operations in 32 bits); with `own` true it
calls the framework.

A case is a dict of plain values:
  op       "window" (attention with a sliding window and sinks, forward),
           "window_train" (the same with its gradients), "write" (quantise
           tokens into the cache and read those rows back), "read" (dequantise a
           cache) or "attend" (attention over the quantised cache)
  B, Hq, Hk, M, N, D   batch, query heads, key/value heads, query (or new)
           tokens, keys (or cache capacity), head dim
  dtype    "fp16" or "bf16"
  window, sinks        0 and 0: causal only ("attend")
  layout   "bhsd": tensors stored (B, H, S, D); "bshd": stored (B, S, H, D) and
           passed as (B, H, S, D) views
  bits     4 or 8: the cache's codes
  ragged   whether the sequences of a batch differ in length
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 32  # channels that share a scale
TOP = {4: 6.0, 8: 448.0}  # largest code
# Exponent bounds of the scales: every code times the largest stays finite in
# the cache's type, the smallest is a normal fp32 number.
EXP_MIN = -126
EXP_MAX = {("fp16", 4): 13, ("fp16", 8): 7, ("bf16", 4): 125, ("bf16", 8): 119}


def _case(op, B, Hq, Hk, M, N, D, dtype, window=0, sinks=0, layout="bhsd", bits=0, ragged=False):
    return {"op": op, "B": B, "Hq": Hq, "Hk": Hk, "M": M, "N": N, "D": D, "dtype": dtype,
            "window": window, "sinks": sinks, "layout": layout, "bits": bits, "ragged": ragged}


def listed():
    named = {
        # One decoding step of a streaming model: one token a sequence against
        # its last 1024 keys and four sinks of a dense cache.
        "window_step": _case("window", 8, 32, 8, 1, 8191, 128, "bf16", 1024, 4),
        # The smallest model the family is run on, one training step.
        "window_train_tiny": _case("window_train", 1, 4, 4, 256, 256, 64, "fp16", 64, 1),
        # A training step of grouped-query heads at the framework's usual length.
        "window_train_4k": _case("window_train", 1, 32, 8, 4096, 4096, 128, "bf16", 1024, 4),
        # A training batch of odd length from a fused QKV projection, no sinks.
        "window_train_ragged": _case("window_train", 2, 12, 12, 1531, 1531, 64, "fp16", 255, 0,
                                     layout="bshd"),
        # Prefill of a long prompt.
        "window_16k": _case("window", 1, 32, 8, 16384, 16384, 128, "bf16", 4096, 64),
        # A decoding step writes one token a sequence.
        "write_step": _case("write", 32, 32, 8, 1, 8192, 128, "bf16", bits=4, ragged=True),
        # A batch of prompts is written after a prefill.
        "write_prompt": _case("write", 4, 32, 8, 4001, 4096, 128, "fp16", bits=8, ragged=True),
        # A cached prompt is handed to an operator that takes dense keys.
        "read_prompt": _case("read", 8, 32, 8, 1, 16384, 128, "bf16", bits=4),
        # Decoding steps: a batch of grouped-query sequences of mixed length, a
        # few very long ones, and many with a window over an 8-bit cache.
        "attend_step": _case("attend", 16, 32, 8, 1, 8191, 128, "bf16", bits=4, ragged=True),
        "attend_long": _case("attend", 4, 32, 8, 1, 131072, 128, "bf16", bits=4),
        "attend_window": _case("attend", 32, 16, 4, 1, 4096, 64, "fp16", 1000, 4, bits=8,
                               ragged=True),
        # A chunk of a prompt against what the cache already holds of it.
        "attend_chunk": _case("attend", 2, 32, 8, 512, 8000, 128, "bf16", bits=4, ragged=True),
    }
    return [{"name": n, **c} for n, c in named.items()]


def _log_int(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi], odd ones among them."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["window", "window_train", "write", "read", "attend", "attend"])
    D = rng.choice([16, 32, 64, 128, 128])
    dtype = rng.choice(["fp16", "bf16"])
    Hk = rng.choice([1, 2, 4, 8])
    G = rng.choice([1, 2, 4, 7, 8]) if op != "window_train" else rng.choice([1, 2, 4, 7])
    if op in ("window", "window_train"):
        N = _log_int(rng, 64, 4096 if op == "window_train" else 8192)
        M = N if op == "window_train" or rng.random() < 0.6 else _log_int(rng, 1, N)
        return _case(op, rng.choice([1, 2]), G * Hk if G * Hk <= 32 else Hk, Hk, M, N, D, dtype,
                     _log_int(rng, 16, 1024), rng.choice([0, 1, 4, 64, 130]),
                     layout=rng.choice(["bhsd", "bshd"]))
    bits = rng.choice([4, 8])
    if op == "write":
        M = _log_int(rng, 1, 4096)
        return _case(op, rng.choice([1, 2, 4]), Hk, Hk, M, M + rng.randrange(0, 200), D, dtype,
                     bits=bits, ragged=rng.random() < 0.5)
    if op == "read":
        return _case(op, rng.choice([1, 3, 8]), Hk, Hk, 1, _log_int(rng, 100, 16384), D, dtype,
                     bits=bits)
    M = 1 if rng.random() < 0.6 else _log_int(rng, 2, 300)
    N = max(M, _log_int(rng, 64, 16384 if M == 1 else 8192))
    window = _log_int(rng, 16, 4096) if rng.random() < 0.4 else 0
    return _case(op, rng.choice([1, 2, 5]) if M > 1 else _log_int(rng, 1, 24),
                 G * Hk if G * Hk <= 32 else Hk, Hk, M, N, D, dtype, window,
                 rng.choice([0, 4, 40]) if window else 0, bits=bits, ragged=rng.random() < 0.7)


def _lengths(case):
    """Keys that each sequence holds (its new tokens among them)."""
    B, M, N = case["B"], case["M"], case["N"]
    if not case["ragged"]:
        return [N] * B
    return [max(M, N - (b * 977) % (N // 2 + 1)) for b in range(B)]


def _counts(case):
    """New tokens of each sequence (the rest of its M rows is padding)."""
    B, M = case["B"], case["M"]
    if not case["ragged"]:
        return [M] * B
    return [M - (b * 131) % (M // 4 + 1) for b in range(B)]


# ---------------------------------------------------------------- inputs


def _normal(gen, shape, dtype, layout="bhsd", channel=False):
    """N(0, 1); channel: key channels of unequal size, as projections give them."""
    B, H, S, D = shape
    x = torch.randn((B, S, H, D) if layout == "bshd" else shape, generator=gen, device="cuda")
    if layout == "bshd":
        x = x.transpose(1, 2)
    if channel:
        x = x * torch.exp(0.5 * torch.randn((1, H, 1, D), generator=gen, device="cuda"))
    return x.to(dtype)


def _steps(y, bits):
    """|x| / s rounded to the grid of the codes, ties to the even code."""
    lo, mant = (0, 1) if bits == 4 else (-6, 3)  # least exponent, mantissa bits
    e = torch.frexp(y)[1] - 1
    step = torch.ldexp(torch.ones_like(y), e.clamp(min=lo) - mant)
    return (torch.round(y / step) * step).clamp(max=TOP[bits])


def _blocks(x):
    D = x.shape[-1]
    return x.reshape(*x.shape[:-1], max(1, D // BLOCK), min(D, BLOCK))


def _quantise(x, dtype, bits):
    """Rounded |x| / s (signed) and the scales' exponents, block by block."""
    y = _blocks(x.float())
    m, e = torch.frexp(y.abs().amax(-1))
    # The top code is 0.75 * 2^3 or 0.875 * 2^9.
    f, t = (0.75, 3) if bits == 4 else (0.875, 9)
    k = torch.where(m == 0, torch.full_like(e, EXP_MIN), e - t + (m > f).to(e.dtype))
    k = k.clamp(EXP_MIN, EXP_MAX[dtype, bits])
    # Two steps, each exact: 2^-k alone can pass fp32's range.
    h = -k // 2
    a = torch.ldexp(torch.ldexp(y.abs(), h[..., None]), (-k - h)[..., None]).clamp(max=TOP[bits])
    return torch.where(y < 0, -_steps(a, bits), _steps(a, bits)), k


def _table(bits, dtype=torch.float32):
    """Values of the codes."""
    vals = []
    for code in range(1 << bits):
        mant = 1 if bits == 4 else 3
        sign = -1.0 if code >> (bits - 1) else 1.0
        mag = code & ((1 << (bits - 1)) - 1)
        e, m = mag >> mant, mag & ((1 << mant) - 1)
        bias = 1 if bits == 4 else 7
        if bits == 8 and mag == 0x7F:
            vals.append(math.nan)
        elif e == 0:
            vals.append(sign * m * 2.0 ** (1 - bias - mant))
        else:
            vals.append(sign * (1 + m / (1 << mant)) * 2.0 ** (e - bias))
    return torch.tensor(vals, dtype=dtype, device="cuda")


def _encode(x, dtype, bits):
    """The cache's bytes of x: codes (two a byte with 4 bits, the lower channel
    in the low half) and biased scale exponents."""
    q, k = _quantise(x, dtype, bits)
    half = 1 << (bits - 1)
    grid = _table(bits)[:half - (1 if bits == 8 else 0)]
    code = torch.searchsorted(grid, q.abs().contiguous()).to(torch.uint8)
    code = (code | (q < 0).to(torch.uint8) * half).reshape(x.shape)
    if bits == 4:
        code = code[..., 0::2] | (code[..., 1::2] << 4)
    return code.contiguous(), (k + 127).to(torch.uint8).contiguous()


def _decode(codes, scales, bits):
    if bits == 4:
        codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    val = _blocks(_table(bits)[codes.long()])
    return torch.ldexp(val, scales.to(torch.int32)[..., None] - 127).flatten(-2)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype, bits = case["op"], DTYPES[case["dtype"]], case["bits"]
    B, Hq, Hk, M, N, D = (case[k] for k in ("B", "Hq", "Hk", "M", "N", "D"))
    st = {"case": case}
    if op in ("window", "window_train"):
        st["q"] = _normal(gen, (B, Hq, M, D), dtype, case["layout"])
        st["k"] = _normal(gen, (B, Hk, N, D), dtype, case["layout"])
        st["v"] = _normal(gen, (B, Hk, N, D), dtype, case["layout"])
        if op == "window_train":
            st["do"] = _normal(gen, (B, Hq, M, D), dtype, case["layout"])
            if own:
                for n in "qkv":
                    st[n].requires_grad_(True)
        return st
    counts = _counts(case)
    st["counts"] = torch.tensor(counts, dtype=torch.int32, device="cuda") if case["ragged"] else None
    if op == "write":
        st["k"] = _normal(gen, (B, Hk, M, D), dtype, channel=True)
        st["v"] = _normal(gen, (B, Hk, M, D), dtype)
        st["start"] = torch.tensor([n - M for n in _lengths(case)], dtype=torch.int32, device="cuda")
        if own:
            from flash_attn_with_score_amd import kv_cache

            st["cache"] = kv_cache.kv_cache(B, Hk, N, D, bits=bits, dtype=dtype, device="cuda")
        return st
    parts = {}
    for n in "kv":
        codes = torch.empty((B, Hk, N, D * bits // 8), dtype=torch.uint8, device="cuda")
        scales = torch.empty((B, Hk, N, max(1, D // BLOCK)), dtype=torch.uint8, device="cuda")
        for b in range(B):
            x = _normal(gen, (1, Hk, N, D), dtype, channel=n == "k")
            c, s = _encode(x, case["dtype"], bits)
            codes[b], scales[b] = c[0], s[0]
        parts[n + "_codes"], parts[n + "_scales"] = codes, scales
    if own:
        from flash_attn_with_score_amd import kv_cache

        st["cache"] = kv_cache.KVCache(**parts, dtype=dtype, bits=bits)
    else:
        st.update(parts)
    if op == "attend":
        st["q"] = _normal(gen, (B, Hq, M, D), dtype)
        st["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    return st


# ---------------------------------------------------------------- plain forms


def _visible(pos, keys, window, sinks):
    ok = keys[None, :] <= pos[:, None]
    if window:
        ok &= (keys[None, :] > pos[:, None] - window) | (keys[None, :] < sinks)
    return ok


def _plain_window(st, train):
    c = st["case"]
    B, Hq, Hk, M, N, D = (c[k] for k in ("B", "Hq", "Hk", "M", "N", "D"))
    q, k, v = st["q"], st["k"], st["v"]
    G, scale = Hq // Hk, D ** -0.5
    ok = _visible(torch.arange(N - M, N, device=q.device), torch.arange(N, device=q.device),
                  c["window"], c["sinks"])
    out = torch.empty((B, Hq, M, D), dtype=q.dtype, device=q.device)
    if train:
        do = st["do"]
        dq, dk, dv = torch.empty_like(out), *(torch.empty((B, Hk, N, D), dtype=q.dtype,
                                                          device=q.device) for _ in "kv")
    for b in range(B):
        for h in range(Hk):
            heads = slice(h * G, (h + 1) * G)
            qf, kf, vf = q[b, heads].float(), k[b, h].float(), v[b, h].float()
            s = (qf @ kf.T) * scale
            s.masked_fill_(~ok, -math.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True))
            p = p / p.sum(-1, keepdim=True)
            o = p @ vf
            out[b, heads] = o.to(q.dtype)
            if train:
                g = do[b, heads].float()
                dv[b, h] = (p.transpose(1, 2) @ g).sum(0).to(q.dtype)
                ds = p * (g @ vf.T - (o * g).sum(-1, keepdim=True))
                dq[b, heads] = ((ds @ kf) * scale).to(q.dtype)
                dk[b, h] = ((ds.transpose(1, 2) @ qf).sum(0) * scale).to(q.dtype)
    return (out, dq, dk, dv) if train else out


def _plain_write(st):
    c = st["case"]
    out = []
    for n in "kv":
        x = st[n]
        q, k = _quantise(x, c["dtype"], c["bits"])
        y = torch.ldexp(q, k[..., None]).flatten(-2)
        if st["counts"] is not None:  # padding rows are not written: the new cache's zeros
            row = torch.arange(c["M"], device=x.device)
            y = torch.where((row[None, :] < st["counts"][:, None])[:, None, :, None], y, 0.0)
        out.append(y.to(x.dtype))
    return tuple(out)


def _plain_read(st):
    c = st["case"]
    return tuple(_decode(st[n + "_codes"], st[n + "_scales"], c["bits"]).to(DTYPES[c["dtype"]])
                 for n in "kv")


def _plain_attend(st):
    c = st["case"]
    B, Hq, Hk, M, N, D = (c[k] for k in ("B", "Hq", "Hk", "M", "N", "D"))
    q, G = st["q"], Hq // Hk
    keys, row = torch.arange(N, device=q.device), torch.arange(M, device=q.device)
    out = torch.empty((B, Hq, M, D), dtype=q.dtype, device=q.device)
    for b in range(B):
        kf = _decode(st["k_codes"][b], st["k_scales"][b], c["bits"])
        vf = _decode(st["v_codes"][b], st["v_scales"][b], c["bits"])
        count = M if st["counts"] is None else st["counts"][b]
        pos = st["lengths"][b] - count + row
        ok = _visible(pos, keys, c["window"], c["sinks"]) & (row < count)[:, None]
        s = (q[b].float().reshape(Hk, G * M, D) @ kf.transpose(1, 2)) * D ** -0.5
        s = s.reshape(Hq, M, N).masked_fill_(~ok, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total == 0, 1.0, total)
        out[b] = (p.reshape(Hk, G * M, N) @ vf).reshape(Hq, M, D).to(q.dtype)
    return out


def run(st):
    c = st["case"]
    op = c["op"]
    if not own:
        if op in ("window", "window_train"):
            return _plain_window(st, op == "window_train")
        return {"write": _plain_write, "read": _plain_read, "attend": _plain_attend}[op](st)
    from flash_attn_with_score_amd import kv_cache
    from flash_attn_with_score_amd.window import attention_window

    if op == "window":
        return attention_window(st["q"], st["k"], st["v"], c["window"], c["sinks"])
    if op == "window_train":
        o = attention_window(st["q"], st["k"], st["v"], c["window"], c["sinks"])
        return (o, *torch.autograd.grad(o, (st["q"], st["k"], st["v"]), st["do"]))
    if op == "write":
        kv_cache.kv_cache_append(st["cache"], st["k"], st["v"], st["start"], st["counts"])
        return kv_cache.kv_cache_read(st["cache"], st["start"], c["M"])
    if op == "read":
        return kv_cache.kv_cache_read(st["cache"])
    return kv_cache.attention_kv_cache(st["q"], st["cache"], st["lengths"], st["counts"],
                                       window=c["window"] or None, sinks=c["sinks"])


# ---------------------------------------------------------------- work


def _row_keys(pos, window, sinks):
    """Keys that a query at this position sees."""
    n = max(0, pos + 1)
    return n if not window else min(n, window) + min(sinks, max(0, n - window))


def _seen(first, last, window, sinks):
    """Keys that at least one query at positions first .. last sees."""
    lo = max(0, first - window + 1) if window else 0
    return max(0, last + 1 - lo) + min(sinks, lo)


def work(case):
    op = case["op"]
    B, Hq, Hk, M, N, D = (case[k] for k in ("B", "Hq", "Hk", "M", "N", "D"))
    w, s = case["window"], case["sinks"]
    row = 0 if not case["bits"] else D * case["bits"] // 8 + max(1, D // BLOCK)
    if op == "write":
        n = Hk * sum(_counts(case))
        # The rows come in, their codes go out and are read again, their
        # values go out (padding rows included).
        return {"bytes": 2 * (n * D * 2 + 2 * n * row + B * Hk * M * D * 2), "flops": 0}
    if op == "read":
        return {"bytes": 2 * B * Hk * N * (row + 2 * D), "flops": 0}
    if op == "attend":
        pairs = keys = 0
        for n, m in zip(_lengths(case), _counts(case)):
            pairs += sum(_row_keys(n - m + i, w, s) for i in range(m))
            keys += _seen(n - m, n - 1, w, s)
        return {"bytes": 2 * B * Hq * M * D * 2 + 2 * Hk * keys * row, "flops": 4 * D * Hq * pairs}
    pairs = B * Hq * sum(_row_keys(N - M + i, w, s) for i in range(M))
    keys = B * Hk * _seen(N - M, N - 1, w, s)
    qo, kv = 2 * B * Hq * M * D * 2, 2 * keys * D * 2
    if op == "window":
        return {"bytes": qo + kv, "flops": 4 * D * pairs}
    # Forward, then dO in and the gradients out; two products and then five.
    return {"bytes": 2 * qo + 2 * B * Hk * N * D * 2 + kv, "flops": 14 * D * pairs}


# ---------------------------------------------------------------- exact


def _exact_attention(q, k, v, pos, window, sinks, do=None, chunk=256):
    """One KV head in 64 bits: q (G, M, D) at positions pos (a list), k, v (N, D).
    Each run of rows takes the keys it can see, sinks and window apart."""
    G, M, D = q.shape
    N = k.shape[0]
    scale = 1.0 / math.sqrt(D)
    o = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for r0 in range(0, M, chunk):
        rows = [r for r in range(r0, min(M, r0 + chunk)) if pos[r] >= 0]
        if not rows:
            continue
        first, last = pos[rows[0]], pos[rows[-1]]
        lo = max(0, first - window + 1) if window else 0
        idx = torch.cat((torch.arange(min(sinks, lo), device=k.device),
                         torch.arange(lo, min(N, last + 1), device=k.device)))
        p0 = torch.tensor([pos[r] for r in rows], device=k.device)
        hidden = idx > p0[:, None]
        if window:
            hidden |= (idx + window <= p0[:, None]) & (idx >= sinks)
        qs, ks, vs = q[:, rows], k[idx], v[idx]
        w = torch.softmax(torch.einsum("gmd,nd->gmn", qs, ks).mul(scale)
                          .masked_fill(hidden, -math.inf), -1)
        o[:, rows] = torch.einsum("gmn,nd->gmd", w, vs)
        if do is not None:
            g = do[:, rows]
            dv.index_add_(0, idx, torch.einsum("gmn,gmd->nd", w, g))
            dp = torch.einsum("gmd,nd->gmn", g, vs)
            ds = w * (dp - (w * dp).sum(-1, keepdim=True)) * scale
            dq[:, rows] = torch.einsum("gmn,nd->gmd", ds, ks)
            dk.index_add_(0, idx, torch.einsum("gmn,gmd->nd", ds, qs))
    return (o, dq, dk, dv) if do is not None else o


def _exact_round(x, dtype, bits):
    """Quantise and read back in 64 bits: the nearest code of the sorted list,
    the even one where two are equally near."""
    C = TOP[bits]
    y = _blocks(x.double())
    amax = y.abs().amax(-1)
    k = torch.ceil(torch.log2(amax.clamp(min=2.0 ** -200) / C))
    k = torch.where(torch.exp2(k - 1) * C >= amax, k - 1, k)
    k = torch.where(torch.exp2(k) * C < amax, k + 1, k)
    s = torch.exp2(k.clamp(EXP_MIN, EXP_MAX[dtype, bits]))[..., None]
    grid = _table(bits, torch.float64)[:(1 << (bits - 1)) - (1 if bits == 8 else 0)]
    mid = (grid[1:] + grid[:-1]) / 2
    a = (y.abs() / s).contiguous()
    below, upto = torch.searchsorted(mid, a), torch.searchsorted(mid, a, right=True)
    code = torch.where(upto % 2 == 0, upto, below)
    return (torch.sign(y) * grid[code] * s).flatten(-2)


def _exact_decode(codes, scales, bits):
    if bits == 4:
        lo, hi = codes.remainder(16), codes.div(16, rounding_mode="floor")
        codes = torch.stack((lo, hi), dim=-1).reshape(*codes.shape[:-1], -1)
    val = _table(bits, torch.float64)[codes.int()]
    per = val.shape[-1] // scales.shape[-1]
    return val * torch.exp2(scales.double() - 127).repeat_interleave(per, -1)


def exact(case, seed):
    st = prepare(case, seed)
    op, bits = case["op"], case["bits"]
    B, Hq, Hk, M, N, D = (case[k] for k in ("B", "Hq", "Hk", "M", "N", "D"))
    G = Hq // Hk
    if op == "write":
        out = []
        for n in "kv":
            y = _exact_round(st[n], case["dtype"], bits)
            for b, m in enumerate(_counts(case)):
                y[b, :, m:] = 0
            out.append(y)
        return tuple(out)
    cache = st.get("cache")
    part = (lambda n: getattr(cache, n)) if cache is not None else (lambda n: st[n])
    if op == "read":
        return tuple(torch.stack([_exact_decode(part(n + "_codes")[b], part(n + "_scales")[b], bits)
                                  for b in range(B)]) for n in "kv")
    train = op == "window_train"
    dev = st["q"].device
    out = [torch.empty((B, Hq, M, D), dtype=torch.float64, device=dev)]
    if train:
        out += [torch.empty((B, h, n, D), dtype=torch.float64, device=dev)
                for h, n in ((Hq, M), (Hk, N), (Hk, N))]
    for b in range(B):
        if op == "attend":
            n, m = _lengths(case)[b], _counts(case)[b]
            pos = [n - m + i if i < m else -1 for i in range(M)]
        else:
            pos = [N - M + i for i in range(M)]
        for h in range(Hk):
            heads = slice(h * G, (h + 1) * G)
            if op == "attend":
                k, v = (_exact_decode(part(n + "_codes")[b, h], part(n + "_scales")[b, h], bits)
                        for n in "kv")
            else:
                k, v = st["k"][b, h].detach().double(), st["v"][b, h].detach().double()
            res = _exact_attention(st["q"][b, heads].detach().double(), k, v, pos, case["window"],
                                   case["sinks"], st["do"][b, heads].double() if train else None)
            if train:
                out[0][b, heads], out[1][b, heads], out[2][b, h], out[3][b, h] = res
            else:
                out[0][b, heads] = res
    return tuple(out) if train else out[0]
