"""The quantised KV cache on the GPU against oracle/cache.py (64 bits).

Codes, scales and read-back values are compared for equality; attention within
the bounds that oracle/cache.py: attend_bounds derives.
"""
from __future__ import annotations

import copy
import math

import pytest
import torch

import flash_attn_with_score_amd as fas
from flash_attn_with_score_amd.kv_cache import (KVCache, attention_kv_cache, kv_cache,
                                                kv_cache_append, kv_cache_read)
from oracle import cache as oracle

pytestmark = pytest.mark.gpu

FP16, BF16 = torch.float16, torch.bfloat16
FORMS = [(d, bits, dt) for d in (16, 32, 64, 128) for bits in (4, 8) for dt in (FP16, BF16)]


def rows(shape, dtype, seed, spread=3.0):
    """Values over several powers of two, as channels of unequal size give them."""
    g = torch.Generator("cpu").manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(spread * torch.randn(*shape[:-1], 1, generator=g))
    return x.clamp(-3e4, 3e4).to(dtype)


def filled(gpu, B, Hk, N, D, bits, dtype, seed, poison=True):
    """A cache whose every row holds quantised values (made by the oracle), and
    those values; poison: bytes that read as NaN wherever nothing is written."""
    k, v = rows((B, Hk, N, D), dtype, seed, 0.3), rows((B, Hk, N, D), dtype, seed + 1, 0.3)
    parts = [t for x in (k, v) for t in oracle.quantise(x, bits)]
    vals = (oracle.decode(*parts[:2], bits), oracle.decode(*parts[2:], bits))
    return KVCache(*(t.to(gpu) for t in parts), dtype=dtype, bits=bits), vals


# ---------------------------------------------------------------- rows in and out


@pytest.mark.parametrize("D,bits,dtype", FORMS)
def test_append_writes_the_nearest_codes(D, bits, dtype, gpu):
    print(f"[case] append D{D} {bits} bits {dtype}", flush=True)
    B, Hk, M, cap = 2, 3, 77, 131
    k, v = rows((B, Hk, M, D), dtype, 1), rows((B, Hk, M, D), dtype, 2)
    # The type's largest values, zeros, halves of a step, and signs of zero.
    big = torch.finfo(dtype).max
    k[0, 0, 0] = big
    k[0, 0, 1] = 0.0
    k[0, 0, 2] = torch.arange(D) % 17 * 0.25 - 2
    k[0, 0, 3] = -0.0
    k[0, 0, 4] = torch.finfo(dtype).smallest_normal
    k[0, 0, 5] = torch.finfo(dtype).smallest_normal * 2.0 ** -3
    v[1, 2, 0, 0] = -big
    cache = kv_cache(B, Hk, cap, D, bits=bits, dtype=dtype, device=gpu)
    start = torch.tensor([5, 54], dtype=torch.int32, device=gpu)
    kv_cache_append(cache, k.to(gpu), v.to(gpu), start)
    gk, gv = kv_cache_read(cache, start, M)
    for n, x, got, codes, scales in (("k", k, gk, cache.k_codes, cache.k_scales),
                                     ("v", v, gv, cache.v_codes, cache.v_scales)):
        want = oracle.quantise(x, bits)
        for b, s in ((0, 5), (1, 54)):
            assert torch.equal(codes[b, :, s:s + M].cpu(), want[0][b]), f"{n} codes of sequence {b}"
            assert torch.equal(scales[b, :, s:s + M].cpu(), want[1][b]), f"{n} scales of sequence {b}"
            assert not codes[b, :, :s].any() and not codes[b, :, s + M:].any(), "other rows changed"
            assert not scales[b, :, :s].any() and not scales[b, :, s + M:].any()
        assert torch.isfinite(got).all()
        assert torch.equal(got.cpu().double(), oracle.decode(*want, bits)), n


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [FP16, BF16])
def test_every_value_of_the_type(bits, dtype, gpu):
    """Each finite value alone in its block (its own scale), and beside a value
    that fixes the scale."""
    print(f"[case] every value {bits} bits {dtype}", flush=True)
    x = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(dtype)
    x = x[torch.isfinite(x)]
    x = x[:x.numel() // 64 * 64]
    alone = torch.zeros(x.numel(), 32, dtype=dtype)
    alone[:, 5] = x
    beside = torch.empty(x.numel() // 16, 32, dtype=dtype)
    beside[:, :16] = x.view(-1, 16)
    beside[:, 16:] = 3.0
    for what, t in (("alone", alone), ("beside", beside)):
        t = t.view(1, 1, -1, 32)
        cache = kv_cache(1, 1, t.shape[2], 32, bits=bits, dtype=dtype, device=gpu)
        kv_cache_append(cache, t.to(gpu), t.to(gpu), 0)
        codes, scales = oracle.quantise(t, bits)
        assert torch.equal(cache.k_codes.cpu(), codes), what
        assert torch.equal(cache.v_scales.cpu(), scales), what
        assert torch.equal(kv_cache_read(cache)[0].cpu().double(), oracle.decode(codes, scales, bits))


@pytest.mark.parametrize("D,bits,dtype", FORMS)
def test_infinities_and_nan_make_their_block_nan(D, bits, dtype, gpu):
    print(f"[case] non-finite D{D} {bits} {dtype}", flush=True)
    x = rows((1, 1, 4, D), dtype, 3, 0.1)
    x[0, 0, 0, 0], x[0, 0, 1, D - 1], x[0, 0, 2, D // 2] = math.inf, -math.inf, math.nan
    cache = kv_cache(1, 1, 4, D, bits=bits, dtype=dtype, device=gpu)
    kv_cache_append(cache, x.to(gpu), x.to(gpu), 0)
    want = oracle.decode(*oracle.quantise(x, bits), bits)
    for got in kv_cache_read(cache):
        assert torch.equal(torch.isnan(got).cpu(), torch.isnan(want))
        assert torch.equal(got.nan_to_num(7).cpu().double(), want.nan_to_num(7))


@pytest.mark.parametrize("D,bits", [(16, 4), (16, 8), (128, 4), (64, 8)])
def test_rows_outside_are_neither_written_nor_read(D, bits, gpu):
    """Starts before and behind the cache, counts that leave rows out, counts past
    the rows given, none at all."""
    print(f"[case] outside D{D} {bits}", flush=True)
    B, Hk, M, cap = 5, 2, 9, 12
    starts, counts = [-4, 7, 0, 2147483640, 3], [9, 20, 4, 9, -1]
    k, v = rows((B, Hk, M, D), BF16, 5), rows((B, Hk, M, D), BF16, 6)
    cache = kv_cache(B, Hk, cap, D, bits=bits, device=gpu)
    start = torch.tensor(starts, dtype=torch.int32, device=gpu)
    kv_cache_append(cache, k.to(gpu), v.to(gpu), start,
                    torch.tensor(counts, dtype=torch.int32, device=gpu))
    codes, scales = oracle.quantise(k, bits)
    want_c, want_s = torch.zeros_like(cache.k_codes.cpu()), torch.zeros_like(cache.k_scales.cpu())
    for b in range(B):
        for i in range(max(0, min(M, counts[b]))):
            r = starts[b] + i
            if 0 <= r < cap:
                want_c[b, :, r], want_s[b, :, r] = codes[b, :, i], scales[b, :, i]
    assert torch.equal(cache.k_codes.cpu(), want_c) and torch.equal(cache.k_scales.cpu(), want_s)
    got = kv_cache_read(cache, start, M)[0].cpu().double()
    vals = oracle.decode(want_c, want_s, bits)
    for b in range(B):
        for i in range(M):
            r = starts[b] + i
            want = vals[b, :, r] if 0 <= r < cap else torch.zeros(Hk, D, dtype=torch.float64)
            assert torch.equal(got[b, :, i], want), (b, i)


def test_strided_rows_and_arrays(gpu):
    """(B, S, H, D) projections, views with odd offsets, and arrays of a larger
    buffer with tokens outermost."""
    print("[case] strides", flush=True)
    B, Hk, M, cap, D, bits = 2, 3, 21, 40, 64, 4
    k = rows((B, M, Hk, D), FP16, 7).transpose(1, 2)
    wide = rows((B, Hk, M, D + 24), FP16, 8)
    v = wide[..., 3:3 + D]  # rows that no vector load can take
    codes = [torch.zeros((cap, B, Hk + 1, 32), dtype=torch.uint8, device=gpu).permute(1, 2, 0, 3)[:, 1:]
             for _ in "kv"]
    scales = [torch.zeros((cap, B, Hk, 4), dtype=torch.uint8, device=gpu)[..., 2:].permute(1, 2, 0, 3)
              for _ in "kv"]
    cache = KVCache(codes[0], scales[0], codes[1], scales[1], dtype=FP16, bits=bits)
    kv_cache_append(cache, k.to(gpu), wide.to(gpu)[..., 3:3 + D], 11)
    for x, got in zip((k, v), kv_cache_read(cache, 11, M)):
        assert torch.equal(got.cpu().double(), oracle.decode(*oracle.quantise(x.contiguous(), bits), bits))


# ---------------------------------------------------------------- attention


def check_attend(gpu, Hq, Hk, M, cap, D, bits, dtype, lengths, counts=None, window=None, sinks=0,
                 sm_scale=None, seed=0, layout="bhsd", edit=None):
    B = len(lengths)
    print(f"[case] attend B{B}H{Hq}K{Hk}M{M}N{cap}D{D} {bits} {dtype} lengths={lengths} "
          f"counts={counts} window={window} sinks={sinks}", flush=True)
    cache, (k, v) = filled(gpu, B, Hk, cap, D, bits, dtype, 10 * seed + 1)
    g = torch.Generator("cpu").manual_seed(10 * seed)
    q = torch.randn((B, M, Hq, D) if layout == "bshd" else (B, Hq, M, D), generator=g).to(dtype)
    q = q.transpose(1, 2) if layout == "bshd" else q
    # What lies behind a sequence reads as NaN.
    for b, n in enumerate(lengths):
        for t in (cache.k_scales, cache.v_scales):
            t[b, :, max(n, 0):] = 255
    if edit is not None:
        edit(cache, k, v)
    gq = q.transpose(1, 2).contiguous().to(gpu).transpose(1, 2) if layout == "bshd" else q.to(gpu)
    as_t = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device=gpu)
    out, lse = attention_kv_cache(gq, cache, as_t(lengths), as_t(counts), window=window, sinks=sinks,
                                  sm_scale=sm_scale, return_log_normalizer=True)
    plain = attention_kv_cache(gq, cache, as_t(lengths), as_t(counts), window=window, sinks=sinks,
                               sm_scale=sm_scale)
    torch.cuda.synchronize()
    assert torch.equal(plain.nan_to_num(9), out.nan_to_num(9)), "the normalizer changes the output"
    out, lse = out.cpu().double(), lse.cpu().double()
    for b in range(B):
        n = max(0, min(lengths[b], cap))
        m = M if counts is None else max(0, min(counts[b], M))
        pos = torch.tensor([n - m + i if i < m else -1 for i in range(M)])
        ref = oracle.attend(q[b], k[b], v[b], pos, window or 0, sinks, sm_scale)
        bound_o, bound_l = oracle.attend_bounds(ref, dtype, D, cap)
        empty = torch.isinf(ref["lse"]) & (ref["lse"] < 0)
        assert (out[b][empty] == 0).all(), "rows that see nothing must be 0"
        assert torch.equal(lse[b] == -math.inf, empty)
        nan_o, nan_l = torch.isnan(ref["out"]), torch.isnan(ref["lse"])
        assert torch.equal(torch.isnan(out[b]), nan_o) and torch.equal(torch.isnan(lse[b]), nan_l)
        err = (out[b] - ref["out"]).abs()
        assert (err <= bound_o)[~nan_o].all(), f"sequence {b}: out off by {err[~nan_o].max():.3e}"
        ok = ~nan_l & ~empty
        assert ((lse[b] - ref["lse"]).abs() <= bound_l)[ok].all(), f"sequence {b}: lse"


@pytest.mark.parametrize("D,bits,dtype", FORMS)
def test_attend_forms(D, bits, dtype, gpu):
    """Each instance: single tokens, and a chunk of more rows than a wave holds."""
    check_attend(gpu, 8, 2, 1, 700, D, bits, dtype, [700, 1, 0, 33, 650], seed=1)
    check_attend(gpu, 4, 2, 40, 300, D, bits, dtype, [300, 40, 41, 7], seed=2)


@pytest.mark.parametrize("M,G", [(1, 1), (1, 7), (1, 32), (1, 33), (2, 16), (3, 8), (32, 1), (33, 1),
                                 (5, 7), (64, 2), (130, 1)])
def test_attend_rows(M, G, gpu):
    """Virtual rows at and around the blocks' edges, ragged sequences and counts."""
    check_attend(gpu, 2 * G, 2, M, 517, 64, 4, BF16, [517, M, 250, 0, 300],
                 [M, M, max(1, M - 1), M, M // 2], seed=3)


@pytest.mark.parametrize("M", [1, 6, 150])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (64, 64), (100, 33), (100, 250),
                                          (5000, 3), (2**40, 2**40)])
def test_attend_window(M, window, sinks, gpu):
    check_attend(gpu, 4, 2, M, 451, 32, 8, FP16, [451, 300, M, 64, 2], [M, M, M, M, min(M, 2)],
                 window=window, sinks=sinks, seed=4)


@pytest.mark.parametrize("M,G", [(1, 4), (40, 2), (300, 1)])
def test_attend_long(M, G, gpu):
    """Enough keys that a row's are dealt to several workgroups, for sequences that
    fill them all, some and one."""
    check_attend(gpu, G, 1, M, 9000, 64, 4, BF16, [9000, 2100, M], None if M > 40 else [M, 1, M],
                 seed=5)
    check_attend(gpu, G, 1, M, 9000, 128, 8, FP16, [8999, 3000], window=2500, sinks=70, seed=6)


@pytest.mark.parametrize("B", [2, 64, 65, 70])
def test_attend_many_sequences(B, gpu):
    """Batches that are and are not dealt by length, most of them short."""
    lengths = [(7 * b * b) % 400 for b in range(B)]
    lengths[1], lengths[-1] = 12000, 5000
    check_attend(gpu, 2, 1, 1, 12000, 32, 4, BF16, lengths, seed=12)
    check_attend(gpu, 3, 1, 2, 12000, 16, 8, FP16, lengths, window=7000, sinks=1, seed=13)


def test_attend_streams_and_graphs(gpu):
    """Calls on two streams at once, and two graphs that share a memory pool,
    replayed in turn: no call sees another's workspace."""
    B, Hq, Hk, cap, D = 2, 8, 2, 9000, 64
    calls = []
    for seed, lens in ((1, [9000, 3]), (2, [4000, 8000])):
        cache, _ = filled(gpu, B, Hk, cap, D, 4, BF16, 40 + seed)
        q = rows((B, Hq, 1, D), BF16, 50 + seed).to(gpu)
        calls.append((q, cache, torch.tensor(lens, dtype=torch.int32, device=gpu)))
    want = [attention_kv_cache(*c) for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = []
    for _ in range(4):
        for c, s in zip(calls, streams):
            with torch.cuda.stream(s):
                got.append(attention_kv_cache(*c))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i % 2]) for i, x in enumerate(got))
    pool, graphs, outs = torch.cuda.graph_pool_handle(), [], []
    for c in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(attention_kv_cache(*c))
        graphs.append(g)
    for _ in range(3):
        for g, x, y in zip(graphs, outs, want):
            x.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(x, y)


def test_attend_scales_and_layouts(gpu):
    check_attend(gpu, 4, 2, 3, 200, 64, 4, FP16, [200, 77], sm_scale=-0.3, seed=7)
    check_attend(gpu, 4, 2, 50, 200, 64, 4, BF16, [200, 77], sm_scale=0.0, layout="bshd", seed=8)
    # Scores that leave no weight but the largest, and lengths past the cache.
    check_attend(gpu, 4, 2, 2, 200, 64, 8, BF16, [1000, -5], sm_scale=8.0, seed=9)


@pytest.mark.parametrize("M", [1, 8, 100])
@pytest.mark.parametrize("D,bits", [(16, 4), (32, 8), (64, 4), (128, 8)])
def test_attend_nan_tokens(M, D, bits, gpu):
    """Tokens that hold NaN reach the rows that see them and no others: behind
    the sequence, in front of the window, and inside a tile that only some rows see."""
    def edit(cache, k, v):
        for t, x, blk in ((cache.v_scales, v, 0), (cache.v_scales, v, v.shape[-1] // 32 - 1),
                          (cache.k_scales, k, 0)):
            for pos in ((250, 120, 90) if x is v else (251, 60)):
                blk = max(0, blk)
                t[:, :, pos, blk] = 255
                x[:, :, pos, 32 * blk:32 * blk + 32] = math.nan

    check_attend(gpu, 4, 2, M, 300, D, bits, BF16, [250, 252, 300, 61], window=90, sinks=5, seed=10,
                 edit=edit)
    check_attend(gpu, 4, 2, M, 300, D, bits, FP16, [300, 251], seed=11, edit=edit)


def test_offsets_past_32_bits(gpu):
    """One head of 2^26 + rows of 64 code bytes: 4 GiB and more behind its first."""
    cap, D = (1 << 26) + 4096, 128
    print("[case] long cache", flush=True)
    arrays = [torch.zeros((1, 1, cap, n), dtype=torch.uint8, device=gpu) for n in (64, 4, 64, 4)]
    cache = KVCache(*arrays, dtype=BF16, bits=4)
    M = 200
    k, v = rows((1, 1, M, D), BF16, 31, 0.3), rows((1, 1, M, D), BF16, 32, 0.3)
    start = cap - M
    kv_cache_append(cache, k.to(gpu), v.to(gpu), start)
    vals = [oracle.decode(*oracle.quantise(x, 4), 4) for x in (k, v)]
    for got, want in zip(kv_cache_read(cache, start, M), vals):
        assert torch.equal(got.cpu().double(), want)
    for rows_q in (1, 60):
        q = torch.randn(1, 1, rows_q, D, generator=torch.Generator("cpu").manual_seed(4)).to(BF16)
        out = attention_kv_cache(q.to(gpu), cache, cap, window=100)
        ref = oracle.attend(q[0], vals[0][0], vals[1][0], torch.arange(M - rows_q, M), 100)
        assert ((out[0].cpu().double() - ref["out"]).abs()
                <= oracle.attend_bounds(ref, BF16, D, 100)[0]).all()


# ---------------------------------------------------------------- together


@pytest.mark.parametrize("bits", [4, 8])
def test_prompt_then_steps(bits, gpu):
    """A padded batch of prompts is written and attended, then tokens follow one by
    one from a captured step; every result equals attention over the values that
    the cache reads back, and the column sums take them too."""
    print(f"[case] prompt and steps {bits}", flush=True)
    B, Hq, Hk, M, cap, D = 3, 8, 2, 70, 100, 64
    counts = [70, 1, 33]
    g = torch.Generator("cpu").manual_seed(0)
    new = lambda h, m: torch.randn(B, h, m, D, generator=g).to(BF16).to(gpu)
    cache = kv_cache(B, Hk, cap, D, bits=bits, device=gpu)
    cnt = torch.tensor(counts, dtype=torch.int32, device=gpu)
    lengths = cnt.clone()
    q, k, v = new(Hq, M), new(Hk, M), new(Hk, M)
    kv_cache_append(cache, k, v, 0, cnt)
    out = attention_kv_cache(q, cache, lengths, cnt)

    def check(q, out, first):
        """Row i of sequence b at position first[b] + i against dense attention."""
        kr, vr = kv_cache_read(cache)
        for b in range(B):
            m = min(q.shape[2], int(lengths[b]) - first[b])
            n = first[b] + m
            dense = fas.attention(q[b:b + 1, :, :m], kr[b:b + 1, :, :n], vr[b:b + 1, :, :n], causal=True)
            absv = fas.attention(q[b:b + 1, :, :m], kr[b:b + 1, :, :n], vr[b:b + 1, :, :n].abs(), causal=True)
            # Both sides are off by at most a rounding of the weights and of the
            # result each (attend_bounds; 1.01: its fp32 terms and absv's own).
            bound = 1.01 * 2 * 2.0 ** -8 * 2 * absv[0].float()
            assert ((out[b, :, :m].float() - dense[0].float()).abs() <= bound + 1e-6).all(), b
            assert not out[b, :, m:].any()

    check(q, out, [0, 0, 0])
    sq, sk, sv = new(Hq, 1), new(Hk, 1), new(Hk, 1)

    def step():
        kv_cache_append(cache, sk, sv, lengths)
        lengths.add_(1)
        return attention_kv_cache(sq, cache, lengths)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(4):
        for t in (sq, sk, sv):
            t.copy_(torch.randn(t.shape, generator=g).to(BF16))
        first = lengths.tolist()
        graph.replay()
        torch.cuda.synchronize()
        assert lengths.tolist() == [n + 1 for n in first]
        eager = attention_kv_cache(sq, cache, lengths)
        assert torch.equal(captured, eager)
        check(sq, captured, first)
    kr, vr = kv_cache_read(cache, 0, 33)
    _, col = fas.attention_with_softmax_col_sum(q[2:, :, :33], kr[2:], vr[2:], causal=True)
    assert abs(float(col.sum()) - Hq * 33) < 1e-2 * Hq * 33


def test_empty_calls(gpu):
    cache = kv_cache(2, 2, 8, 32, device=gpu)
    none = torch.empty(2, 2, 0, 32, dtype=BF16, device=gpu)
    kv_cache_append(cache, none, none, 8)
    assert kv_cache_read(cache, 8, 0)[0].shape == (2, 2, 0, 32)
    assert attention_kv_cache(torch.empty(2, 4, 0, 32, dtype=BF16, device=gpu), cache, 8).shape == (2, 4, 0, 32)
    nothing = kv_cache(2, 2, 0, 32, device=gpu)
    out, lse = attention_kv_cache(torch.ones(2, 4, 3, 32, dtype=BF16, device=gpu), nothing, 0,
                                  return_log_normalizer=True)
    assert not out.any() and (lse == -math.inf).all()
    empty = kv_cache(0, 2, 8, 32, device=gpu)
    assert attention_kv_cache(torch.ones(0, 4, 3, 32, dtype=BF16, device=gpu), empty, 8).shape[0] == 0


def test_refusals(gpu):
    cache = kv_cache(2, 2, 8, 32, device=gpu)
    x = torch.ones(2, 2, 3, 32, dtype=BF16, device=gpu)
    q = torch.ones(2, 4, 1, 32, dtype=BF16, device=gpu)
    i32 = lambda n: torch.zeros(n, dtype=torch.int32, device=gpu)
    for bad in (-1, 6):
        with pytest.raises(ValueError):
            kv_cache_append(cache, x, x, bad)
        with pytest.raises(ValueError):
            kv_cache_read(cache, bad, 3)
    with pytest.raises(ValueError):
        kv_cache_read(cache, 0, -1)
    for bad in (-1, 9):
        with pytest.raises(ValueError):
            attention_kv_cache(q, cache, bad)
    for kw in ({"window": 0}, {"window": -3}, {"window": 4, "sinks": -1}):
        with pytest.raises(ValueError):
            attention_kv_cache(q, cache, 8, **kw)
    with pytest.raises(AssertionError):
        attention_kv_cache(q, cache, 8, sinks=2)
    for bad in (i32(3), i32(2).long(), i32(2).view(1, 2)):
        with pytest.raises(AssertionError):
            kv_cache_append(cache, x, x, bad)
        with pytest.raises(AssertionError):
            attention_kv_cache(q, cache, bad)
        with pytest.raises(AssertionError):
            attention_kv_cache(q, cache, 8, bad)
    with pytest.raises(AssertionError):
        attention_kv_cache(q, cache, 8, 1)
    with pytest.raises(RuntimeError):
        attention_kv_cache(q, cache, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(AssertionError):
        kv_cache_append(cache, x.half(), x, 0)
    with pytest.raises(AssertionError):
        kv_cache_append(cache, x, x[:, :, :2], 0)
    with pytest.raises(AssertionError):
        kv_cache_append(cache, x[..., :16], x[..., :16], 0)
    with pytest.raises(RuntimeError):
        kv_cache_append(cache, x.cpu(), x, 0)
    with pytest.raises(AssertionError):
        attention_kv_cache(q.half(), cache, 8)
    with pytest.raises(AssertionError):
        attention_kv_cache(q[:, :3], cache, 8)
    with pytest.raises(AssertionError):
        attention_kv_cache(q[:1], cache, 8)
    with pytest.raises(RuntimeError):
        attention_kv_cache(q.cpu(), cache, 8)
    with pytest.raises(RuntimeError, match="sm_scale"):
        attention_kv_cache(q, cache, 8, sm_scale=math.inf)
    c, s = cache.k_codes, cache.k_scales
    for parts in ((c, s, c, s[:, :, :7]), (c, s, c[..., :8], s), (c.short(), s, c, s), (c, s, c[0], s)):
        with pytest.raises(AssertionError):
            KVCache(*parts, dtype=BF16, bits=4)
    with pytest.raises(AssertionError):
        KVCache(c, s, c, s, dtype=torch.float32, bits=4)
    with pytest.raises(AssertionError):
        KVCache(c, s, c, s, dtype=BF16, bits=5)
    wide = torch.zeros((2, 2, 8, 24), dtype=torch.uint8, device=gpu)[..., 4:20]
    with pytest.raises(TypeError):
        attention_kv_cache(q, cache, 2.5)
    shared = KVCache(*(t[:1].expand(2, -1, -1, -1) for t in (c, s, cache.v_codes, cache.v_scales)),
                     dtype=BF16, bits=4)
    with pytest.raises(RuntimeError, match="repeat"):
        kv_cache_append(shared, x, x, 0)
    with pytest.raises(RuntimeError, match="share"):
        kv_cache_append(KVCache(c, s, c, s, dtype=BF16, bits=4), x, x, 0)
    with pytest.raises(RuntimeError, match="aligned"):
        kv_cache_append(KVCache(wide, s, c, s, dtype=BF16, bits=4), x, x, 0)


def test_copies_and_shared_prompts(gpu):
    """A copied or pickled cache has arrays of its own; sequences may share a
    cache that is not appended to; rows expanded over tokens and heads are taken."""
    print("[case] copies", flush=True)
    B, Hk, M, D = 3, 2, 50, 64
    cache = kv_cache(B, Hk, 64, D, device=gpu)
    row = torch.randn(D, generator=torch.Generator("cpu").manual_seed(1)).to(BF16).to(gpu)
    x = row.expand(B, Hk, M, D)
    kv_cache_append(cache, x, x, 0)
    twin = copy.deepcopy(cache)
    kv_cache_append(twin, torch.zeros_like(x), torch.zeros_like(x), 0)
    for y in kv_cache_read(cache, 0, M):
        want = oracle.decode(*oracle.quantise(row.cpu()[None], 4), 4)[0]
        assert torch.equal(y.cpu().double(), want.expand(B, Hk, M, D))
    assert all((y == 0).all() for y in kv_cache_read(twin, 0, M))
    y = torch.randn(B, Hk, M, D, generator=torch.Generator("cpu").manual_seed(2)).to(BF16).to(gpu)
    kv_cache_append(cache, y, y.flip(2), 0)
    shared = KVCache(*(t[1:2].expand(B, -1, -1, -1) for t in
                       (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)), dtype=BF16, bits=4)
    q = torch.randn(B, 4, 2, D, generator=torch.Generator("cpu").manual_seed(3)).to(BF16).to(gpu)
    got = attention_kv_cache(q, shared, M)
    for b in range(B):
        one = KVCache(*(t[1:2] for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)),
                      dtype=BF16, bits=4)
        assert torch.equal(got[b:b + 1], attention_kv_cache(q[b:b + 1].contiguous(), one, M))
    qx = q[:, :, :1].expand(B, 4, 5, D)
    assert torch.equal(attention_kv_cache(qx, cache, M), attention_kv_cache(qx.contiguous(), cache, M))
