"""attention_window on the GPU, forward and backward, against oracle/window.py
(64 bits) within the bounds derived there."""
from __future__ import annotations

import math

import pytest
import torch

import flash_attn_with_score_amd as fas
from flash_attn_with_score_amd.window import attention_window
from oracle import inputs, window as oracle

pytestmark = pytest.mark.gpu

FP16, BF16 = torch.float16, torch.bfloat16


def check(gpu, B, Hq, Hk, M, N, D, dtype, window, sinks, grad=True, layout="bhsd", sm_scale=None,
          seed=0, scale=1.0, few_keys=False):
    print(f"[case] window B{B}H{Hq}K{Hk}M{M}N{N}D{D} {dtype} window={window} sinks={sinks} "
          f"grad={grad} {layout}", flush=True)
    q, k, v = inputs.make_qkv(B, Hq, Hk, M, N, D, dtype=dtype, seed=seed, scale=scale)
    do = torch.randn(B, Hq, M, D, generator=torch.Generator("cpu").manual_seed(seed + 1)).to(dtype)
    lay = (lambda x: x.transpose(1, 2).contiguous().to(gpu).transpose(1, 2)) if layout == "bshd" \
        else (lambda x: x.to(gpu))
    gq, gk, gv, gdo = (lay(x) for x in (q, k, v, do))
    for x in (gq, gk, gv):
        x.requires_grad_(grad)
    out, lse = attention_window(gq, gk, gv, window, sinks, sm_scale=sm_scale,
                                return_log_normalizer=True)
    got = {"out": out.detach(), "lse": lse}
    if grad:
        got.update(zip(("dq", "dk", "dv"), torch.autograd.grad(out, (gq, gk, gv), gdo)))
    else:
        assert torch.equal(attention_window(gq, gk, gv, window, sinks, sm_scale=sm_scale), out)
    torch.cuda.synchronize()
    for b in range(B):
        ref = oracle.reference(q[b], k[b], v[b], min(window, 1 << 40), min(sinks, 1 << 40),
                               do[b] if grad else None, sm_scale, few_keys)
        empty = torch.isinf(ref["lse"])
        assert torch.equal(got["lse"][b].cpu() == -math.inf, empty)
        assert (got["out"][b].cpu()[empty] == 0).all()
        for n, x in got.items():
            x, want = x[b].cpu().double(), ref[n]
            if n == "lse":
                x, want = torch.where(empty, 0.0, x), torch.where(empty, 0.0, want)
            assert torch.isfinite(x).all(), n
            over = ((x - want).abs() / ref[n + "_bound"]).max().item() if x.numel() else 0.0
            assert over <= 1.0, f"{n} of entry {b}: {over:.3f} times its bound"


@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", [FP16, BF16])
def test_instances(D, dtype, gpu):
    check(gpu, 2, 4, 2, 300, 300, D, dtype, 70, 5, seed=D)


@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("M,N,window,sinks", [(128, 128, 500, 0), (90, 100, 80, 4), (120, 100, 200, 1),
                                              (500, 500, 100, 28), (300, 410, 64, 64), (333, 333, 1, 0)])
def test_rows_of_few_keys(M, N, window, sinks, D, gpu):
    """No block's first row sees more than 128 keys: out's rounding does not reach
    the gradients."""
    check(gpu, 1, 4, 2, M, N, D, (FP16, BF16)[D % 128 == 0], window, sinks, seed=M + D, few_keys=True)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 200), (31, 0), (32, 32), (33, 31),
                                          (64, 1), (65, 64), (127, 129), (128, 0), (200, 65),
                                          (411, 3), (412, 0), (2**50, 2**50), (2**70, 2**70)])
def test_masks(window, sinks, gpu):
    """Windows and sinks at and around the tiles' edges, up to the causal mask."""
    check(gpu, 1, 2, 1, 411, 411, 64, BF16, window, sinks, seed=3)


@pytest.mark.parametrize("M,N", [(1, 1), (1, 500), (1, 64), (33, 33), (128, 129), (7, 700), (200, 333),
                                 (300, 100), (129, 1), (257, 256)])
@pytest.mark.parametrize("window,sinks", [(50, 4), (1000, 0)])
def test_lengths(M, N, window, sinks, gpu):
    """Single tokens, queries behind a prefix, and more queries than keys (rows that
    see nothing)."""
    check(gpu, 1, 4, 2, M, N, 32, FP16, window, sinks, seed=4)


@pytest.mark.parametrize("Hq,Hk", [(1, 1), (7, 1), (6, 2), (16, 1), (5, 5)])
def test_heads_and_layouts(Hq, Hk, gpu):
    check(gpu, 2, Hq, Hk, 190, 190, 64, BF16, 60, 4, layout="bshd", seed=5)


@pytest.mark.parametrize("sm_scale", [-0.2, 0.0, 3.0])
def test_scales(sm_scale, gpu):
    check(gpu, 1, 4, 2, 150, 150, 64, FP16, 40, 2, sm_scale=sm_scale, seed=6)


def test_long_windows_split(gpu):
    """Few rows over many keys (several workgroups a row), and long runs of rows
    behind sinks (several workgroups a key block)."""
    check(gpu, 1, 4, 2, 1, 6000, 128, BF16, 5000, 4, seed=7)
    check(gpu, 2, 8, 8, 3, 4001, 64, FP16, 1500, 70, grad=False, seed=8)
    check(gpu, 1, 2, 1, 2100, 2100, 64, BF16, 90, 130, seed=9)
    check(gpu, 1, 4, 4, 1500, 1700, 128, FP16, 129, 1, seed=10)


@pytest.mark.parametrize("D", [16, 64, 128])
@pytest.mark.parametrize("dtype", [FP16, BF16])
def test_key_blocks_dealt_to_several_workgroups(D, dtype, gpu):
    """Sinks that all later rows see beside short windows: parts of key blocks, runs
    over several blocks and heads, blocks that no row sees."""
    check(gpu, 2, 4, 2, 1300, 1300, D, dtype, 40, 130, seed=21)
    check(gpu, 1, 2, 2, 900, 2100, D, dtype, 129, 33, seed=22)
    check(gpu, 1, 6, 1, 700, 500, D, dtype, 33, 1, seed=23)


@pytest.mark.parametrize("D,dtype", [(32, FP16), (64, BF16), (128, FP16), (128, BF16)])
def test_scores_of_hundreds(D, dtype, gpu):
    """Rows whose maximum rises from tile to tile, and weights that vanish."""
    check(gpu, 1, 4, 2, 300, 300, D, dtype, 150, 4, seed=24, scale=6.0)
    check(gpu, 1, 4, 2, 2, 1100, D, dtype, 900, 4, seed=25, scale=6.0)


def test_window_past_the_keys_is_causal_attention(gpu):
    q, k, v = (t.to(gpu) for t in inputs.make_qkv(2, 4, 2, 333, 333, 128, dtype=FP16, seed=11))
    out, lse = attention_window(q, k, v, 333, return_log_normalizer=True)
    want, L, *_ = fas.attention(q, k, v, causal=True, return_log_normalizer=True)
    ref = oracle.reference(q[0].cpu(), k[0].cpu(), v[0].cpu(), 333)
    # Both sides are within the bound of the exact result.
    assert ((out[0] - want[0]).cpu().double().abs() <= 2 * ref["out_bound"]).all()
    assert (lse - L).abs().max() < 1e-3


def test_unaligned_and_broadcast_inputs(gpu):
    """Rows that start off 16 bytes are copied; an expanded K gets its gradient
    summed over what it was expanded to; an expanded dO is taken as it is."""
    B, H, M, D = 2, 4, 100, 32
    wide = torch.randn(B, H, M, D + 8, generator=torch.Generator("cpu").manual_seed(1)).to(BF16)
    q = wide.to(gpu)[..., 3:3 + D].requires_grad_(True)
    k1 = wide[:1, :1, :, :D].to(gpu).requires_grad_(True)
    k = k1.expand(B, H, M, D)
    v = wide[..., 8:].contiguous().to(gpu).requires_grad_(True)
    out = attention_window(q, k, v, 30, 2)
    gq, gk, gv = torch.autograd.grad(out.sum(), (q, k1, v))
    do = torch.ones(H, M, D, dtype=BF16)
    refs = [oracle.reference(q[b].detach().cpu(), k[b].detach().cpu(), v[b].detach().cpu(), 30, 2, do)
            for b in range(B)]
    for b, ref in enumerate(refs):
        assert ((gq[b].cpu().double() - ref["dq"]).abs() <= ref["dq_bound"]).all()
        assert ((gv[b].cpu().double() - ref["dv"]).abs() <= ref["dv_bound"]).all()
    want = sum(r["dk"].sum(0) for r in refs)
    # Torch adds B * H rounded gradients: half a step of the running sum each.
    bound = sum(r["dk_bound"].sum(0) + 2.0 ** -8 * r["dk"].abs().sum(0) * B * H for r in refs)
    assert ((gk[0, 0].cpu().double() - want).abs() <= bound).all()


def test_gradients_of_token_sums(gpu):
    """A dO that is expanded over the tokens, as a sum over them hands it on."""
    B, H, M, D = 1, 4, 90, 64
    q, k, v = (x.to(gpu).requires_grad_(True) for x in inputs.make_qkv(B, H, H, M, M, D, dtype=FP16, seed=4))
    w = torch.randn(B, H, D, generator=torch.Generator("cpu").manual_seed(5)).to(FP16).to(gpu)
    out = attention_window(q, k, v, 40, 1)
    got = torch.autograd.grad(out, (q, k, v), w[:, :, None].expand(B, H, M, D), retain_graph=True)
    want = torch.autograd.grad(out, (q, k, v), w[:, :, None].expand(B, H, M, D).contiguous())
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_second_derivatives_are_refused(gpu):
    q, k, v = (x.to(gpu).requires_grad_(True) for x in inputs.make_qkv(1, 2, 2, 40, 40, 32, dtype=FP16, seed=4))
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(attention_window(q, k, v, 16).sum(), q, create_graph=True)


def test_captured_training_step(gpu):
    """Forward and backward in one graph; every replay equals the eager step."""
    B, H, Hk, M, D = 1, 4, 2, 260, 64
    print("[case] captured window step", flush=True)
    q, k, v = (t.to(gpu).requires_grad_(True)
               for t in inputs.make_qkv(B, H, Hk, M, M, D, dtype=BF16, seed=1))
    do = torch.randn(B, H, M, D, generator=torch.Generator("cpu").manual_seed(9)).to(BF16).to(gpu)

    def step(q, k, v):
        o = attention_window(q, k, v, 70, 3)
        return (o, *torch.autograd.grad(o, (q, k, v), do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(q, k, v)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step(q, k, v)
    for seed in (2, 3, 4):
        fresh = inputs.make_qkv(B, H, Hk, M, M, D, dtype=BF16, seed=seed)
        with torch.no_grad():
            for dst, src in zip((q, k, v), fresh):
                dst.copy_(src.to(gpu))
        graph.replay()
        torch.cuda.synchronize()
        eager = step(*(t.detach().clone().requires_grad_(True) for t in (q, k, v)))
        torch.cuda.synchronize()
        for name, x, y in zip(("o", "dq", "dk", "dv"), static, eager):
            assert torch.equal(x, y), f"{name}, inputs seed {seed}"
    del graph


@pytest.mark.parametrize("other", [lambda x: fas.attention(x, x, x, causal=True), lambda x: x * 2])
def test_capture_beside_another_operators_graph_is_refused(other, gpu):
    print("[case] captured window step beside another operator's graph", flush=True)
    q, k, v = (t.to(gpu).requires_grad_(True)
               for t in inputs.make_qkv(1, 2, 2, 130, 130, 32, dtype=BF16, seed=1))
    alive = other(k)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph of the same leaves"):
        with torch.cuda.graph(graph):
            out = attention_window(q, k, v, 50, 1)
            torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
    out = alive = None
    torch.cuda.synchronize()
    want = torch.autograd.grad(attention_window(q, k, v, 50, 1), (q, k, v), torch.ones_like(q))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attention_window(q, k, v, 50, 1)
        first = torch.autograd.grad(out, (q, k, v), torch.ones_like(out), retain_graph=True)
        again = attention_window(k, q, v, 50, 1)  # (leaves of this capture's own graph)
        torch.autograd.grad(again, (q, k, v), torch.ones_like(out))
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(first, want))
    del graph


def test_capture_beside_an_eager_graph_is_refused(gpu):
    """A captured backward pass while an eager graph of the same leaves lives would
    end the process in the autograd engine: it raises, and the step can be
    captured once the eager graph is gone."""
    print("[case] captured window step beside an eager graph", flush=True)
    q, k, v = (t.to(gpu).requires_grad_(True)
               for t in inputs.make_qkv(1, 2, 1, 130, 130, 32, dtype=BF16, seed=1))
    alive = attention_window(q, k, v, 50, 1)
    want = torch.autograd.grad(alive, (q, k, v), torch.ones_like(alive), retain_graph=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph of the same leaves"):
        with torch.cuda.graph(graph):
            out = attention_window(q, k, v, 50, 1)
            torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
    out = alive = None
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attention_window(q, k, v, 50, 1)
        got = torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    del graph


def test_other_streams(gpu):
    """Two calls on two streams at once: nothing is shared between them."""
    args = [[t.to(gpu) for t in inputs.make_qkv(1, 8, 2, 4, 5000, 64, dtype=FP16, seed=s)] for s in (1, 2)]
    want = [attention_window(*a, 3000, 4) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    got = []
    for _ in range(3):
        for a, s in zip(args, streams):
            with torch.cuda.stream(s):
                got.append(attention_window(*a, 3000, 4))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert torch.equal(g, want[i % 2])


def test_empty_calls(gpu):
    e = lambda *s: torch.zeros(*s, dtype=FP16, device=gpu).requires_grad_(True)
    for B, M, N in ((0, 3, 3), (1, 0, 5), (1, 5, 0)):
        q, k, v = e(B, 2, M, 32), e(B, 2, N, 32), e(B, 2, N, 32)
        out = attention_window(q, k, v, 4)
        assert out.shape == q.shape and not out.any()
        for x, g in zip((q, k, v), torch.autograd.grad(out, (q, k, v), torch.ones_like(out))):
            assert g.shape == x.shape and not g.any()


def test_refusals(gpu):
    q, k, v = (t.to(gpu) for t in inputs.make_qkv(1, 4, 2, 8, 8, 32, dtype=FP16, seed=0))
    for window, sinks in ((0, 0), (-1, 0), (4, -1)):
        with pytest.raises(ValueError):
            attention_window(q, k, v, window, sinks)
    with pytest.raises(AssertionError):
        attention_window(q, k[:, :, :, :16], v, 4)
    with pytest.raises(AssertionError):
        attention_window(q.float(), k.float(), v.float(), 4)
    with pytest.raises(AssertionError):
        attention_window(q, k, v[:, :, :7], 4)
    with pytest.raises(AssertionError):
        attention_window(q[:, :3], k, v, 4)
    with pytest.raises(RuntimeError):
        attention_window(q.cpu(), k, v, 4)
    with pytest.raises(RuntimeError, match="sm_scale"):
        attention_window(q, k, v, 4, sm_scale=math.nan)
