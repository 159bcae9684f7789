"""Windowed attention and the quantised KV cache, without a GPU: the C ABI's
refusals (sent with addresses that nothing dereferences), workspace sizes,
records, the Python launchers' checks, and the 64-bit oracle against finite
differences and the definition."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from flash_attn_with_score_amd import _native, kv_cache
from flash_attn_with_score_amd.window import attention_window
from oracle import cache as oracle_cache, window as oracle_window

PTR = 0x1000000  # 256-byte aligned
SIZE_MAX = ctypes.c_size_t(-1).value


@pytest.fixture(scope="module")
def lib():
    return _native.load()


def untyped(lib, name, *args):
    """The entry point with NULL where the declared types want an array."""
    fn = getattr(ctypes.CDLL(lib._name), name)
    fn.argtypes = None
    return fn(*(ctypes.c_void_p(a) if a is None else a for a in args))


P = ctypes.c_void_p(PTR)


def attn_args(B=1, Hq=4, Hk=2, M=300, N=300, D=64, causal=1, dtype=1):
    a = _native.AttnArgs()
    a.dtype, a.causal, a.sm_scale = dtype, causal, D ** -0.5
    a.batch, a.heads_q, a.heads_k, a.seqlen_q, a.seqlen_k, a.head_dim = B, Hq, Hk, M, N, D
    a.q = a.k = a.v = a.out = PTR
    for name, H, L in (("q_stride", Hq, M), ("k_stride", Hk, N), ("v_stride", Hk, N),
                       ("out_stride", Hq, M)):
        setattr(a, name, _native._I64x4(H * L * D, L * D, D, 1))
    return a


def cache_args(B=2, H=2, N=100, D=64, bits=4, dtype=1):
    """(Keys and values at one address: an append of it is refused.)"""
    c = _native.KVCacheArgs()
    c.dtype, c.bits, c.batch, c.heads, c.capacity, c.head_dim = dtype, bits, B, H, N, D
    code, scale = D * bits // 8, max(1, D // 32)
    for n in "kv":
        for part, row in (("codes", code), ("scales", scale)):
            setattr(c, f"{n}_{part}", PTR)
            setattr(c, f"{n}_{part}_stride", _native._I64x3(H * N * row, N * row, row))
    return c


def query_args(c, Hq=4, M=3, lengths=0, lengths_all=50, window=0, sinks=0):
    q = _native.KVQueryArgs()
    D = c.head_dim
    q.heads_q, q.tokens, q.q, q.out = Hq, M, PTR, PTR
    q.q_stride = q.out_stride = _native._I64x4(Hq * M * D, M * D, D, 1)
    q.lengths, q.lengths_all, q.window, q.sinks, q.sm_scale = lengths, lengths_all, window, sinks, 0.125
    return q


def refused(lib, rc, code, *words):
    assert rc == code, (rc, _native.last_error(lib))
    msg = _native.last_error(lib)
    for w in words:
        assert w in msg, (w, msg)


# ---------------------------------------------------------------- window


def window_call(lib, a, window=16, sinks=0, lse=PTR, ws=PTR, nbytes=None, lst=(300 * 4, 300, 1)):
    if nbytes is None:
        nbytes = lib.fas_attention_window_workspace(ctypes.byref(a), window, sinks, 0)
        nbytes = 0 if nbytes == SIZE_MAX else nbytes
    return lib.fas_attention_window(ctypes.byref(a), window, sinks, lse, _native._I64x3(*lst), ws,
                                    nbytes, None)


def backward_call(lib, a, window=16, sinks=0, nbytes=None, lse=PTR, **null):
    if nbytes is None:
        nbytes = lib.fas_attention_window_workspace(ctypes.byref(a), window, sinks, 1)
    g = lambda n: null.get(n, PTR)
    return lib.fas_attention_window_backward(
        ctypes.byref(a), window, sinks, g("dout"), a.q_stride, lse, _native._I64x3(1200, 300, 1),
        g("dq"), a.q_stride, g("dk"), a.k_stride, g("dv"), a.k_stride, PTR, nbytes, None)


@pytest.mark.parametrize("change,code,word", [
    (dict(causal=0), _native.FAS_ERR_INVALID, "causal"),
    (dict(D=48), _native.FAS_ERR_UNSUPPORTED, "head_dim"),
    (dict(dtype=3), _native.FAS_ERR_UNSUPPORTED, "dtype"),
    (dict(Hq=3), _native.FAS_ERR_INVALID, "multiple"),
    (dict(M=1 << 27, Hq=8), _native.FAS_ERR_UNSUPPORTED, "sizes"),
])
def test_window_refuses_shapes(lib, change, code, word):
    a = attn_args(**change)
    assert lib.fas_attention_window_workspace(ctypes.byref(a), 16, 0, 0) == SIZE_MAX
    assert lib.fas_attention_window_workspace(ctypes.byref(a), 16, 0, 1) == SIZE_MAX
    refused(lib, window_call(lib, a), code, "fas_attention_window", word)
    refused(lib, backward_call(lib, a, nbytes=0), code, "fas_attention_window_backward", word)


def test_window_refuses_arguments(lib):
    a = attn_args()
    for window, sinks in ((0, 0), (-5, 0), (4, -1)):
        refused(lib, window_call(lib, a, window, sinks), _native.FAS_ERR_INVALID, "window")
    a.dropout_p = 0.1
    refused(lib, window_call(lib, a), _native.FAS_ERR_UNSUPPORTED, "dropout")
    for name in ("q", "k", "v", "out"):
        a = attn_args()
        setattr(a, name, None)
        refused(lib, window_call(lib, a), _native.FAS_ERR_INVALID, name + " is NULL")
        a = attn_args()
        setattr(a, name, PTR + 2)
        refused(lib, window_call(lib, a), _native.FAS_ERR_INVALID, name, "aligned")
    refused(lib, window_call(lib, attn_args(), lst=(-1, 300, 1)), _native.FAS_ERR_INVALID, "lse")
    refused(lib, untyped(lib, "fas_attention_window", ctypes.byref(attn_args()), ctypes.c_int64(16),
                         ctypes.c_int64(0), P, None, None, ctypes.c_size_t(0), None),
            _native.FAS_ERR_INVALID, "lse")
    for name in ("dout", "dq", "dk", "dv"):
        refused(lib, backward_call(lib, attn_args(), **{name: None}), _native.FAS_ERR_INVALID, name)
    refused(lib, backward_call(lib, attn_args(), lse=None), _native.FAS_ERR_INVALID, "lse")
    need = lib.fas_attention_window_workspace(ctypes.byref(attn_args()), 16, 0, 1)
    assert need > 0
    refused(lib, backward_call(lib, attn_args(), nbytes=need - 1), _native.FAS_ERR_WORKSPACE, str(need))
    few = attn_args(M=1, N=100000)
    need = lib.fas_attention_window_workspace(ctypes.byref(few), 50000, 0, 0)
    assert need > 0
    refused(lib, window_call(lib, few, 50000, ws=None), _native.FAS_ERR_WORKSPACE, str(need))
    refused(lib, window_call(lib, few, 50000, ws=PTR + 16), _native.FAS_ERR_WORKSPACE)


def test_window_workspace_grows_with_what_is_split(lib):
    size = lambda back, window=1024, sinks=4, **kw: lib.fas_attention_window_workspace(
        ctypes.byref(attn_args(**kw)), window, sinks, back)
    assert size(0, B=1, Hq=32, Hk=32, M=4096, N=4096) == 0  # enough row blocks
    # One token over a long cache: fp32 parts of at most 512 workgroups' rows.
    assert 0 < size(0, M=1, N=1 << 20, window=1 << 20) <= 2 * 512 * 32 * (64 + 2) * 4 + 1024
    # Two fp32 numbers a padded row, and at most two slabs for each of 512 workgroups.
    rows = 2 * 32 * 4096 * 4
    assert rows <= size(1, Hq=32, Hk=8, M=4096, N=4096, D=128) <= rows + 264 * 2 * 128 * 256 * 4


def test_window_empty_calls_launch_nothing(lib):
    for kw in (dict(B=0), dict(M=0)):
        assert window_call(lib, attn_args(**kw)) == 0
    assert backward_call(lib, attn_args(B=0)) == 0


# ---------------------------------------------------------------- cache


def move(lib, c, append=True, M=5, start=None, start_all=0, counts=None, k=PTR, stride=None):
    st = stride or _native._I64x4(c.heads * M * c.head_dim, M * c.head_dim, c.head_dim, 1)
    if append:
        return lib.fas_kv_cache_append(ctypes.byref(c), k, st, PTR, st, M, start, start_all, counts, None)
    return lib.fas_kv_cache_read(ctypes.byref(c), k, st, PTR, st, M, start, start_all, None)


def attend(lib, c, q, ws=PTR, nbytes=None, lse=None, lst=(0, 0, 0)):
    if nbytes is None:
        nbytes = lib.fas_attention_kv_cache_workspace(ctypes.byref(c), ctypes.byref(q))
        nbytes = 0 if nbytes == SIZE_MAX else nbytes
    return lib.fas_attention_kv_cache(ctypes.byref(c), ctypes.byref(q), lse, _native._I64x3(*lst), ws, nbytes, None)


@pytest.mark.parametrize("change,code,word", [
    (dict(bits=5), _native.FAS_ERR_UNSUPPORTED, "bits"),
    (dict(D=48), _native.FAS_ERR_UNSUPPORTED, "head_dim"),
    (dict(dtype=2), _native.FAS_ERR_UNSUPPORTED, "dtype"),
    (dict(B=-1), _native.FAS_ERR_INVALID, "size"),
    (dict(H=0), _native.FAS_ERR_INVALID, "size"),
    (dict(N=(1 << 28) + 1), _native.FAS_ERR_UNSUPPORTED, "sizes"),
    (dict(B=1 << 20, H=1 << 5), _native.FAS_ERR_UNSUPPORTED, "sizes"),
])
def test_cache_refuses_forms(lib, change, code, word):
    c = cache_args(**change)
    for rc in (move(lib, c), move(lib, c, False), attend(lib, c, query_args(c))):
        refused(lib, rc, code, word)
    assert lib.fas_attention_kv_cache_workspace(ctypes.byref(c), ctypes.byref(query_args(c))) == SIZE_MAX


def test_cache_refuses_arrays(lib):
    for n in ("k_codes", "k_scales", "v_codes", "v_scales"):
        for append in (True, False):
            c = cache_args()
            setattr(c, n, None)
            refused(lib, move(lib, c, append), _native.FAS_ERR_INVALID, n + " is NULL")
        c = cache_args()
        setattr(c, n, PTR + 1)
        refused(lib, attend(lib, c, query_args(c)), _native.FAS_ERR_INVALID, n, "aligned")
        for bad, code in (((-64, 64, 64), _native.FAS_ERR_INVALID), ((64, 1 << 47, 64), _native.FAS_ERR_INVALID),
                          ((64, 64, 0), _native.FAS_ERR_INVALID), ((64, 64, 1 << 32), _native.FAS_ERR_UNSUPPORTED)):
            c = cache_args()
            setattr(c, n + "_stride", _native._I64x3(*bad))
            refused(lib, move(lib, c), code, n)


def test_cache_refuses_rows(lib):
    c = cache_args(N=100)
    for start, M in ((-1, 5), (96, 5), (0, 101), (1 << 40, 5)):
        for append in (True, False):
            refused(lib, move(lib, c, append, M, start_all=start), _native.FAS_ERR_INVALID, "outside")
    refused(lib, move(lib, c, M=-1), _native.FAS_ERR_INVALID, "tokens")
    refused(lib, move(lib, c, start=PTR, M=(1 << 28) + 1), _native.FAS_ERR_UNSUPPORTED, "sizes")
    refused(lib, move(lib, c, start=PTR + 2), _native.FAS_ERR_INVALID, "start")
    refused(lib, move(lib, c, counts=PTR + 1), _native.FAS_ERR_INVALID, "counts")
    refused(lib, move(lib, c, k=None), _native.FAS_ERR_INVALID, "k is NULL")
    refused(lib, move(lib, c, stride=_native._I64x4(0, 0, 63, 1)), _native.FAS_ERR_INVALID, "k")
    n5, zero = ctypes.c_int64(5), ctypes.c_int64(0)
    refused(lib, untyped(lib, "fas_kv_cache_append", ctypes.byref(c), P, None, P, None, n5, None, zero, None, None),
            _native.FAS_ERR_INVALID, "strides")
    st = _native._I64x4(0, 0, 64, 1)
    refused(lib, untyped(lib, "fas_kv_cache_read", None, P, st, P, st, n5, None, zero, None),
            _native.FAS_ERR_INVALID, "cache is NULL")


def test_append_refuses_rows_in_one_place(lib):
    for n in ("k_codes", "v_scales"):
        for at in (0, 1):
            c = cache_args()
            row = 32 if "codes" in n else 2
            st = [200 * row, 100 * row, row]
            st[at] = 0
            setattr(c, n + "_stride", _native._I64x3(*st))
            for part in ("codes", "scales"):  # distinct otherwise
                setattr(c, "v_" + part, PTR + (1 << 30))
            refused(lib, move(lib, c), _native.FAS_ERR_INVALID, "repeat")
    refused(lib, move(lib, cache_args()), _native.FAS_ERR_INVALID, "share")
    c = cache_args()
    c.v_codes = PTR + (1 << 30)
    refused(lib, move(lib, c), _native.FAS_ERR_INVALID, "share")


def test_attention_refuses_queries(lib):
    c = cache_args()
    for change, code, word in ((dict(Hq=3), _native.FAS_ERR_INVALID, "multiple"),
                               (dict(M=-1), _native.FAS_ERR_INVALID, "size"),
                               (dict(M=1 << 28), _native.FAS_ERR_UNSUPPORTED, "sizes"),
                               (dict(window=-1), _native.FAS_ERR_INVALID, "window"),
                               (dict(sinks=-1), _native.FAS_ERR_INVALID, "sinks"),
                               (dict(lengths_all=101), _native.FAS_ERR_INVALID, "length"),
                               (dict(lengths_all=-1), _native.FAS_ERR_INVALID, "length")):
        q = query_args(c, **change)
        refused(lib, attend(lib, c, q), code, word)
    for name, v in (("q", None), ("out", None), ("lengths", PTR + 2), ("counts", PTR + 3)):
        q = query_args(c)
        setattr(q, name, v)
        refused(lib, attend(lib, c, q), _native.FAS_ERR_INVALID, name)
    q = query_args(c)
    q.sm_scale = math.inf
    refused(lib, attend(lib, c, q), _native.FAS_ERR_INVALID, "sm_scale")
    refused(lib, attend(lib, c, query_args(c), lse=PTR, lst=(-1, 3, 1)), _native.FAS_ERR_INVALID, "lse")
    refused(lib, untyped(lib, "fas_attention_kv_cache", ctypes.byref(c), None, None, None, None,
                         ctypes.c_size_t(0), None), _native.FAS_ERR_INVALID, "query is NULL")
    big = cache_args(N=1 << 20)
    q = query_args(big, lengths=PTR, M=1)
    need = lib.fas_attention_kv_cache_workspace(ctypes.byref(big), ctypes.byref(q))
    assert need > 0
    refused(lib, attend(lib, big, q, nbytes=need - 1), _native.FAS_ERR_WORKSPACE, str(need))
    refused(lib, attend(lib, big, q, ws=None), _native.FAS_ERR_WORKSPACE)


def test_cache_empty_calls_launch_nothing(lib):
    c = cache_args(B=0)
    assert move(lib, c) == 0 and move(lib, c, False) == 0 and attend(lib, c, query_args(c)) == 0
    c = cache_args()
    assert move(lib, c, M=0) == 0 and attend(lib, c, query_args(c, M=0)) == 0


def test_launchers_refuse_host_tensors():
    q, k = torch.zeros(1, 2, 4, 32, dtype=torch.float16), torch.zeros(1, 2, 4, 32, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="HIP device"):
        attention_window(q, k, k, 4)
    for D in (48, 256):
        x = torch.zeros(1, 2, 4, D, dtype=torch.float16)
        with pytest.raises(AssertionError):
            attention_window(x, x, x, 4)
    codes, scales = torch.zeros(1, 2, 4, 16, dtype=torch.uint8), torch.zeros(1, 2, 4, 1, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="HIP device"):
        kv_cache.KVCache(codes, scales, codes, scales, dtype=torch.float16, bits=4)
    with pytest.raises(RuntimeError, match="HIP device"):
        kv_cache.kv_cache(1, 2, 4, 32, device="cpu")
    for kw in ({"head_dim": 48}, {"head_dim": 32, "bits": 3}):
        with pytest.raises(AssertionError):
            kv_cache.kv_cache(1, 2, 4, **kw, device="cpu")


# ---------------------------------------------------------------- oracle


@pytest.mark.parametrize("window,sinks", [(3, 0), (4, 2), (100, 0), (1, 1)])
def test_gradients_against_differences(window, sinks):
    """oracle/window.py's gradients against central differences of its output, in
    64 bits: truncation h^2 times a third derivative of order one, and rounding
    2^-52 / h, both far below 1e-6."""
    g = torch.Generator("cpu").manual_seed(1)
    Hq, Hk, M, N, D, h = 4, 2, 7, 9, 16, 1e-4
    q, k, v, do = (torch.randn(s, generator=g, dtype=torch.float64)
                   for s in ((Hq, M, D), (Hk, N, D), (Hk, N, D), (Hq, M, D)))

    def loss(q, k, v):
        x = (q, k, v)
        see = oracle_cache.visible(torch.arange(N - M, N), N, window, sinks)
        s = (x[0] @ x[1].repeat_interleave(Hq // Hk, 0).transpose(1, 2)) / math.sqrt(D)
        p = torch.softmax(s.masked_fill(~see, -math.inf), -1)
        return float((p @ x[2].repeat_interleave(Hq // Hk, 0) * do).sum())

    ref = oracle_window.reference(q, k, v, window, sinks, do)
    for name, t in (("dq", q), ("dk", k), ("dv", v)):
        for idx in [(0, 0, 0), (1, 3, 5), (1, 6, 15), (0, 2, 7)]:
            a, b = t.clone(), t.clone()
            a[idx] += h
            b[idx] -= h
            args = {"dq": (a, k, v), "dk": (q, a, v), "dv": (q, k, a)}[name]
            brgs = {"dq": (b, k, v), "dk": (q, b, v), "dv": (q, k, b)}[name]
            num = (loss(*args) - loss(*brgs)) / (2 * h)
            assert abs(num - float(ref[name][idx])) < 1e-6, (name, idx)


@pytest.mark.parametrize("bits", [4, 8])
def test_oracle_codes(bits):
    """Every code decodes to its definition; quantising a decoded row gives the
    same values back; halves round to the even code."""
    D = 32
    codes = torch.arange(1 << bits, dtype=torch.int64)
    sign, mant, bias = 1 << (bits - 1), (1, 3)[bits == 8], (1, 7)[bits == 8]
    mag = codes % sign
    e, m = mag >> mant, mag & ((1 << mant) - 1)
    val = torch.where(e == 0, m * 2.0 ** (1 - bias - mant),
                      (1 + m / 2.0 ** mant) * torch.exp2((e - bias).double()))
    val = torch.where(codes >= sign, -val, val)
    rows = codes.reshape(-1, D) if bits == 8 else torch.cat((codes, codes)).reshape(1, D)
    raw = rows if bits == 8 else rows[:, 0::2] + 16 * rows[:, 1::2]
    got = oracle_cache.decode(raw.to(torch.uint8), torch.full((rows.shape[0], 1), 127, dtype=torch.uint8), bits)
    want = val[rows]
    if bits == 8:
        assert torch.isnan(got[want.abs() == 480]).all()
        got, want = got[want.abs() < 480], want[want.abs() < 480]
    assert torch.equal(got, want.double())
    x = torch.randn(50, 64, generator=torch.Generator("cpu").manual_seed(3)).to(torch.bfloat16)
    once = oracle_cache.decode(*oracle_cache.quantise(x, bits), bits)
    again = oracle_cache.decode(*oracle_cache.quantise(once.to(torch.bfloat16), bits), bits)
    assert torch.equal(once, again)
    step = 2.0 if bits == 4 else 32.0  # of the largest codes
    top = oracle_cache.TOP[bits]
    x = torch.zeros(1, 32, dtype=torch.bfloat16)
    x[0, 0], x[0, 1], x[0, 2] = top, top - step / 2, top - 3 * step / 2
    got = oracle_cache.decode(*oracle_cache.quantise(x, bits), bits)[0]
    # Codes of the top value are even in 8 bits (126), odd in 4 (7).
    assert got[1] == (top if bits == 8 else top - step)
