"""attention_window: causal attention with a sliding window and sinks, with its
backward pass.

No counterpart in the reference, whose masks are none or causal.  A query sees
the last `window` keys up to its own and the first `sinks` keys of the sequence,
which stay visible behind the window.  The forward and backward kernels visit
the tiles of visible keys alone, so the work grows with window + sinks and not
with the sequence; kv_cache.attention_kv_cache is the same mask over a quantised
cache.
"""
from __future__ import annotations

import math
import operator

import torch

from . import _common, _native
from .flash import _check_inputs

__all__ = ["attention_window", "WindowAttention"]

# Any window or sinks past every sequence length mean the same.
_MOST = 1 << 62


def _workspace(args: bytes, window: int, sinks: int, backward: int, device):
    name = "fas_attention_window_workspace"
    nbytes = _native.fast(name)(args, window, sinks, backward)
    ptr, buf = _common.allocate_workspace(name, nbytes, device)
    return ptr, nbytes, buf


# The autograd engine hands a leaf's gradient over to the stream on which the
# leaf's accumulation node was made.  While an eager graph of the same leaf lives
# that node is the eager one, and in a captured backward pass the hand-over
# draws a stream that is not captured into the capture, which ends the process
# (seen with torch 2.10 on ROCm: a segmentation fault at the capture's end).
# So the nodes carry their stream, and such a backward pass raises instead.
_STREAM = "flash_attn_with_score_amd.stream"


def _mark_leaves(out) -> None:
    stream = None
    for node, _ in out.grad_fn.next_functions:
        if type(node).__name__ == "AccumulateGrad":
            if stream is None:
                stream = _common.current_raw_stream(out.device.index)
            node.metadata.setdefault(_STREAM, stream)


def _mark_strangers(*inputs) -> None:
    """Before a captured forward: leaves whose accumulation nodes other operators'
    graphs hold, on a stream that cannot be asked for, get no stream at all.  (A
    node that nothing holds goes, with its mark, when the reference here does.)"""
    for x in inputs:
        if x.requires_grad and x.is_leaf:
            node = torch.autograd.graph.get_gradient_edge(x).node
            node.metadata.setdefault(_STREAM, None)
            del node


def _check_capture(ctx, device) -> None:
    if not torch.cuda.is_current_stream_capturing():
        return
    stream = _common.current_raw_stream(device.index)
    for node, _ in ctx.next_functions:
        if type(node).__name__ == "AccumulateGrad" and node.metadata.get(_STREAM, stream) != stream:
            raise RuntimeError(
                "flash_attn_with_score_amd: attention_window's backward is captured while an eager "
                "graph of the same leaves lives; drop its outputs before the capture")


def _forward(q, k, v, window, sinks, sm_scale, want_lse):
    """(q, k, v as the kernels take them, out, normalizer or None)."""
    q, k, v = _common.as_row_operand(q), _common.as_row_operand(k), _common.as_row_operand(v)
    o = _common.new_output(q)
    L = torch.empty(q.shape[:3], device=q.device, dtype=torch.float32) if want_lse else None
    args = _native.pack_args(q, k, v, o, True, sm_scale)
    ws_ptr, ws_bytes, ws = _workspace(args, window, sinks, 0, q.device)
    _common.call("fas_attention_window", q, args, window, sinks,
                 0 if L is None else L.data_ptr(), None if L is None else _native.pack_strides(L),
                 ws_ptr, ws_bytes)
    return q, k, v, o, L


class WindowAttention(torch.autograd.Function):
    """fas_attention_window and fas_attention_window_backward."""

    @staticmethod
    def forward(ctx, q, k, v, window, sinks, sm_scale, return_log_normalizer):
        q, k, v, o, L = _forward(q, k, v, window, sinks, sm_scale, True)
        ctx.save_for_backward(q, k, v, o, L)
        ctx.window, ctx.sinks, ctx.sm_scale = window, sinks, sm_scale
        if return_log_normalizer:
            ctx.mark_non_differentiable(L)
            return o, L
        return o

    @staticmethod
    def backward(ctx, do, *ignored):
        if torch.is_grad_enabled():
            raise RuntimeError("flash_attn_with_score_amd: attention_window is differentiable once "
                               "(create_graph=True)")
        q, k, v, o, L = ctx.saved_tensors
        _check_capture(ctx, q.device)
        do = _common.as_row_operand(do)
        dq, dk, dv = _common.new_output(q), _common.new_output(k), _common.new_output(v)
        args = _native.pack_args(q, k, v, o, True, ctx.sm_scale)
        ws_ptr, ws_bytes, ws = _workspace(args, ctx.window, ctx.sinks, 1, q.device)
        _common.call("fas_attention_window_backward", q, args, ctx.window, ctx.sinks, do.data_ptr(),
                     _native.pack_strides(do), L.data_ptr(), _native.pack_strides(L), dq.data_ptr(),
                     _native.pack_strides(dq), dk.data_ptr(), _native.pack_strides(dk), dv.data_ptr(),
                     _native.pack_strides(dv), ws_ptr, ws_bytes)
        return dq, dk, dv, None, None, None, None


def attention_window(q, k, v, window: int, sinks: int = 0, sm_scale: float | None = None,
                     return_log_normalizer: bool = False):
    """Attention of q (B, Hq, M, D) over k, v (B, Hk, N, D), Hq % Hk == 0: query row
    i, at position p = (N - M) + i, sees key j iff j <= p and (j > p - window or
    j < sinks).

    Returns out like q, or (out, log_normalizer (B, Hq, M) fp32, which is not
    differentiable).  Rows that see no key (M > N) are 0, their normalizer -inf.
    Differentiable once in q, k and v; like attention(), it takes finite inputs: a
    hidden key has weight 0, and 0 times an infinity or NaN in it is NaN."""
    _check_inputs(q, k, v)
    _common.check_device_inputs(q, k, v, 0.0)
    if window < 1:
        raise ValueError(f"flash_attn_with_score_amd: window {window} must be at least 1")
    if sinks < 0:
        raise ValueError(f"flash_attn_with_score_amd: sinks {sinks} must not be negative")
    window, sinks = min(operator.index(window), _MOST), min(operator.index(sinks), _MOST)
    sm_scale = 1.0 / math.sqrt(q.shape[3]) if sm_scale is None else float(sm_scale)
    if not (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)):
        *_, out, L = _forward(q, k, v, window, sinks, sm_scale, return_log_normalizer)
        return (out, L) if return_log_normalizer else out
    if torch.cuda.is_current_stream_capturing():
        _mark_strangers(q, k, v)
    res = WindowAttention.apply(q, k, v, window, sinks, sm_scale, return_log_normalizer)
    _mark_leaves(res[0] if return_log_normalizer else res)
    return res
