"""A quantised KV cache: written row by row, read back, attended over.

No counterpart in the reference, whose launchers take dense fp16 or bf16 keys
and values.  The cache holds codes of 4 bits (e2m1) or 8 bits (e4m3) with a
power-of-two scale per block of 32 channels: 4.25 or 8.25 bits a value instead
of 16.  kv_cache_append quantises rows as they are written, kv_cache_read gives
them back as values, which every entry point of this package takes as k and v
(the column sums of a cached prompt, say), and attention_kv_cache is attention
over the codes themselves, for decoding and for chunks of a prompt.

Numbers that belong to the sequences of a batch (`start`, `lengths`, `counts`)
are an int for all of them, or an int32 device tensor of `batch` elements that
the kernels read when they run: nothing synchronises, and a captured call
follows the tensor's contents.  What an int says is checked here; what a tensor
says is bounded on the device (rows outside the cache are not written, lengths
and counts are clamped to what there is).

Calls on a cache are ordered like any work on its tensors: by stream.  None of
them is differentiable.
"""
from __future__ import annotations

import math
import operator
from dataclasses import dataclass, field

import torch

from . import _common, _native

__all__ = ["KVCache", "kv_cache", "kv_cache_append", "kv_cache_read", "attention_kv_cache"]

BLOCK = 32  # channels that share a scale


@dataclass(frozen=True, eq=False)
class KVCache:
    """The cache's four uint8 arrays: codes (batch, heads_k, capacity, head_dim *
    bits / 8) and scales (batch, heads_k, capacity, max(1, head_dim / 32)) of the
    keys and of the values, the type of the values and the bits of a code.  An
    array's rows must be contiguous and aligned to their size (up to 16 bytes);
    its other strides are free (only a cache that is not appended to may repeat
    rows, a prompt that its sequences share, say).  The arrays' memory has to stay
    where it is.  include/fas.h says what the bytes mean."""

    k_codes: torch.Tensor
    k_scales: torch.Tensor
    v_codes: torch.Tensor
    v_scales: torch.Tensor
    dtype: torch.dtype
    bits: int
    head_dim: int = field(init=False)
    batch: int = field(init=False)
    heads_k: int = field(init=False)
    capacity: int = field(init=False)
    device: torch.device = field(init=False)
    _record: bytes = field(init=False, repr=False)

    def __post_init__(self):
        arrays = (self.k_codes, self.k_scales, self.v_codes, self.v_scales)
        assert self.dtype in _native.DTYPE_CODES, \
            f"dtype must be float16 or bfloat16, got {self.dtype}"
        assert self.bits in (4, 8), f"bits must be 4 or 8, got {self.bits}"
        assert all(t.dtype == torch.uint8 and t.dim() == 4 for t in arrays), \
            "codes and scales must be 4-dimensional uint8 tensors"
        if not all(t.is_cuda for t in arrays):
            raise RuntimeError("flash_attn_with_score_amd: codes and scales must be HIP device tensors")
        assert all(t.device == self.k_codes.device for t in arrays), \
            "codes and scales must be on one device"
        B, H, N, nbytes = self.k_codes.shape
        D = nbytes * 8 // self.bits
        assert D in _common.SUPPORTED_HEAD_DIMS, f"head_dim must be one of 16, 32, 64, 128, got {D}"
        blocks = max(1, D // BLOCK)
        assert self.v_codes.shape == self.k_codes.shape, "k_codes and v_codes must have one shape"
        assert self.k_scales.shape == self.v_scales.shape == (B, H, N, blocks), \
            f"scales must be {(B, H, N, blocks)}"
        assert all(t.stride(3) == 1 or t.shape[3] == 1 for t in arrays), "rows must be contiguous"
        record = _native.pack_kv_cache(*arrays, self.dtype, self.bits, D)
        for name, value in (("head_dim", D), ("batch", B), ("heads_k", H), ("capacity", N),
                            ("device", self.k_codes.device), ("_record", record)):
            object.__setattr__(self, name, value)

    def __reduce__(self):  # a copy has arrays, and so addresses, of its own
        return (KVCache, (self.k_codes, self.k_scales, self.v_codes, self.v_scales, self.dtype, self.bits))


def kv_cache(batch: int, heads_k: int, capacity: int, head_dim: int, bits: int = 4,
             dtype: torch.dtype = torch.bfloat16, device=None) -> KVCache:
    """An empty cache (all values zero) for `capacity` tokens of each sequence."""
    assert head_dim in _common.SUPPORTED_HEAD_DIMS, \
        f"head_dim must be one of 16, 32, 64, 128, got {head_dim}"
    assert bits in (4, 8), f"bits must be 4 or 8, got {bits}"
    device = torch.device("cuda") if device is None else device
    codes = (batch, heads_k, capacity, head_dim * bits // 8)
    scales = (batch, heads_k, capacity, max(1, head_dim // BLOCK))
    return KVCache(*(torch.zeros(s, dtype=torch.uint8, device=device)
                     for s in (codes, scales, codes, scales)), dtype=dtype, bits=bits)


def _per_sequence(name: str, x, cache: KVCache):
    """(tensor or None, int) of a per-sequence number."""
    if not isinstance(x, torch.Tensor):
        return None, operator.index(x)
    assert x.dtype == torch.int32 and x.shape == (cache.batch,), \
        f"{name} must be an int or an int32 tensor of {cache.batch} elements"
    if not x.is_cuda:
        raise RuntimeError(f"flash_attn_with_score_amd: {name} must be a HIP device tensor")
    assert x.device == cache.device, f"{name} must be on the cache's device"
    return (x if x.stride(0) == 1 else x.contiguous()), 0


def _counts(counts, cache: KVCache):
    """Tensor or None of the rows of each sequence; None: all of them."""
    if counts is None:
        return None
    assert isinstance(counts, torch.Tensor), "counts must be None or an int32 tensor"
    return _per_sequence("counts", counts, cache)[0]


def _ptr(x) -> int:
    return 0 if x is None else x.data_ptr()


def _span(name: str, first: int, rows: int, cache: KVCache) -> None:
    if not 0 <= first <= cache.capacity - rows:
        raise ValueError(f"flash_attn_with_score_amd: {name}: rows [{first}, {first + rows}) lie "
                         f"outside the cache of {cache.capacity}")


def kv_cache_append(cache: KVCache, k: torch.Tensor, v: torch.Tensor, start, counts=None) -> None:
    """Quantises k and v (batch, heads_k, M, head_dim) into the cache: row i of
    sequence b becomes cache row start[b] + i, for i < counts[b] (None: all M).
    No other row of the cache changes.

    A block of 32 channels gets the least power-of-two scale that clips none of
    its values (the largest of the type excepted, include/fas.h), and its values
    round to the nearest code, ties to even; a block that holds an infinity or
    NaN reads back as NaN."""
    shape = k.shape
    assert shape == v.shape and len(shape) == 4 and \
        (shape[0], shape[1], shape[3]) == (cache.batch, cache.heads_k, cache.head_dim), \
        f"k and v must be {cache.batch} x {cache.heads_k} x M x {cache.head_dim}, " \
        f"got {tuple(k.shape)}, {tuple(v.shape)}"
    assert k.dtype == cache.dtype and v.dtype == cache.dtype, f"k and v must be {cache.dtype}"
    if not (k.is_cuda and v.is_cuda):
        raise RuntimeError("flash_attn_with_score_amd: k and v must be HIP device tensors")
    assert k.device == cache.device and v.device == cache.device, "k and v must be on the cache's device"
    M = shape[2]
    start_t, start_all = _per_sequence("start", start, cache)
    counts_t = _counts(counts, cache)
    if start_t is None:
        _span("kv_cache_append", start_all, M, cache)
    k, v = _common.as_row_operand(k), _common.as_row_operand(v)
    _common.call("fas_kv_cache_append", cache.k_codes, cache._record, k.data_ptr(),
                 _native.pack_strides(k), v.data_ptr(), _native.pack_strides(v), M, _ptr(start_t),
                 start_all, _ptr(counts_t))


def kv_cache_read(cache: KVCache, start=0, length: int | None = None):
    """Cache rows start[b] .. start[b] + length - 1 as (k, v), each (batch, heads_k,
    length, head_dim) in the cache's type, exactly what the codes stand for;
    length None: up to the capacity, from an int `start`.  With a tensor `start`,
    rows outside the cache read as zeros."""
    start_t, start_all = _per_sequence("start", start, cache)
    if length is None:
        assert start_t is None, "a tensor start needs a length"
        length = cache.capacity - start_all
    if length < 0:
        raise ValueError(f"flash_attn_with_score_amd: kv_cache_read: length {length}")
    if start_t is None:
        _span("kv_cache_read", start_all, length, cache)
    shape = (cache.batch, cache.heads_k, length, cache.head_dim)
    k = torch.empty(shape, dtype=cache.dtype, device=cache.device)
    v = torch.empty_like(k)
    strides = _native.pack_strides(k)
    _common.call("fas_kv_cache_read", cache.k_codes, cache._record, k.data_ptr(), strides,
                 v.data_ptr(), strides, length, _ptr(start_t), start_all)
    return k, v


def attention_kv_cache(q: torch.Tensor, cache: KVCache, lengths, counts=None,
                       window: int | None = None, sinks: int = 0, sm_scale: float | None = None,
                       return_log_normalizer: bool = False):
    """Attention of each sequence's last tokens over its cached keys.

    q (batch, Hq, M, head_dim), Hq a multiple of the cache's heads; lengths:
    keys that each sequence holds, those of q's tokens among them (append
    first); counts: how many of q's rows are real, the first ones (None: all M).
    Row i of sequence b is at position lengths[b] - counts[b] + i and sees key j
    iff j <= position and, with a window, (j > position - window or j < sinks).

    Returns out like q, or (out, log_normalizer (batch, Hq, M) fp32).  Rows
    past counts, and rows that see no key, are 0 (their normalizer -inf).
    Cache rows past a sequence's length do not influence it."""
    assert q.dim() == 4 and q.shape[0] == cache.batch and q.shape[3] == cache.head_dim, \
        f"q must be {cache.batch} x Hq x M x {cache.head_dim}, got {tuple(q.shape)}"
    B, H, M, D = q.shape
    assert H % cache.heads_k == 0, "number of heads in q must be a multiple of the cache's"
    assert q.dtype == cache.dtype, f"q must be {cache.dtype}"
    if not q.is_cuda:
        raise RuntimeError("flash_attn_with_score_amd: q must be a HIP device tensor")
    assert q.device == cache.device, "q must be on the cache's device"
    if window is None:
        assert sinks == 0, "sinks need a window"
        window = 0
    elif window < 1:
        raise ValueError(f"flash_attn_with_score_amd: window {window} must be at least 1")
    if sinks < 0:
        raise ValueError(f"flash_attn_with_score_amd: sinks {sinks} must not be negative")
    lengths_t, lengths_all = _per_sequence("lengths", lengths, cache)
    counts_t = _counts(counts, cache)
    if lengths_t is None and not 0 <= lengths_all <= cache.capacity:
        raise ValueError(f"flash_attn_with_score_amd: length {lengths_all} lies outside "
                         f"[0, {cache.capacity}]")
    q = _common.as_row_operand(q)
    out = _common.new_output(q)
    lse = torch.empty((B, H, M), dtype=torch.float32, device=q.device) if return_log_normalizer \
        else None
    query = _native.pack_kv_query(q, out, lengths_t, lengths_all, counts_t, int(window), int(sinks),
                                  float(1.0 / math.sqrt(D) if sm_scale is None else sm_scale))
    nbytes = _native.fast("fas_attention_kv_cache_workspace")(cache._record, query)
    ws_ptr, ws = _common.allocate_workspace("fas_attention_kv_cache_workspace", nbytes, q.device)
    _common.call("fas_attention_kv_cache", q, cache._record, query, _ptr(lse),
                 None if lse is None else _native.pack_strides(lse), ws_ptr, nbytes)
    return (out, lse) if return_log_normalizer else out
