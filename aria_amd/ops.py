"""Host-pointer op surface of the MI355X backend, mirroring the reference's
src/aria_ops.h and src/aria_quant.h names and argument meaning (numpy in, numpy
out). Each call goes through the C ABI (aria_cuda_* of include/aria_gpu.h or
aria_hip_* of include/aria_hip.h): copy in, run the gfx950 kernel, copy out.

In-place ops of the reference (silu, gelu_tanh, softcap, softmax, rope_apply)
return a new array and leave the argument untouched here.
"""
from __future__ import annotations

import numpy as np

from . import check, lib


def _p(a):
    return None if a is None else a.ctypes.data


def _f32(a):
    if a is None:
        return None
    a = np.ascontiguousarray(a, dtype=np.float32)
    return a


# ---- aria_gpu.h wrappers (src/aria_gpu.h:38-61) ----

def rmsnorm(x, w, eps):
    x = _f32(x); w = _f32(w)
    dim = x.shape[-1]
    y = np.empty_like(x)
    lib().aria_cuda_rmsnorm(_p(y), _p(x), _p(w), x.size // dim, dim, eps)
    return y


def gemma_rmsnorm(x, w, eps):
    x = _f32(x); w = _f32(w)
    dim = x.shape[-1]
    y = np.empty_like(x)
    lib().aria_cuda_gemma_rmsnorm(_p(y), _p(x), _p(w), x.size // dim, dim, eps)
    return y


def dynamic_tanh(x, alpha, w, b):
    x = _f32(x); w = _f32(w); b = _f32(b)
    dim = x.shape[-1]
    y = np.empty_like(x)
    lib().aria_cuda_dynamic_tanh(_p(y), _p(x), alpha, _p(w), _p(b), x.size // dim, dim)
    return y


def softcap(x, cap):
    y = _f32(x).copy()
    lib().aria_cuda_softcap(_p(y), y.size, cap)
    return y


def silu(x):
    y = _f32(x).copy()
    lib().aria_cuda_silu(_p(y), y.size)
    return y


def gelu_tanh(x):
    y = _f32(x).copy()
    lib().aria_cuda_gelu_tanh(_p(y), y.size)
    return y


def silu_gate(gate, up):
    gate = _f32(gate); up = _f32(up)
    out = np.empty_like(gate)
    lib().aria_cuda_silu_gate(_p(out), _p(gate), _p(up), gate.size)
    return out


def softmax(x, mask=None):
    y = _f32(x).copy()
    mask = _f32(mask)
    cols = y.shape[-1]
    lib().aria_cuda_softmax(_p(y), y.size // cols, cols, _p(mask))
    return y


def rope_apply(x, cos_t, sin_t, rot_dim):
    y = _f32(x).copy()
    cos_t = _f32(cos_t); sin_t = _f32(sin_t)
    N, D = y.shape[-2], y.shape[-1]
    lib().aria_cuda_rope_apply(_p(y), _p(cos_t), _p(sin_t), y.size // (N * D), N, D, rot_dim)
    return y


def linear(x, W, b=None):
    x = _f32(x); W = _f32(W); b = _f32(b)
    M, K = x.shape
    N = W.shape[0]
    y = np.empty((M, N), np.float32)
    lib().aria_cuda_linear(_p(y), _p(x), _p(W), _p(b), M, K, N)
    return y


def matmul(A, B):
    A = _f32(A); B = _f32(B)
    M, K = A.shape
    N = B.shape[1]
    Cm = np.empty((M, N), np.float32)
    lib().aria_cuda_matmul(_p(Cm), _p(A), _p(B), M, K, N)
    return Cm


def attention(q, k, v, mask=None):
    q = _f32(q); k = _f32(k); v = _f32(v); mask = _f32(mask)
    H, Nq, D = q.shape
    Nk = k.shape[1]
    out = np.empty_like(q)
    lib().aria_cuda_attention(_p(out), _p(q), _p(k), _p(v), H, Nq, Nk, D, _p(mask))
    return out


def conv1d(inp, w, bias, pad):
    inp = _f32(inp); w = _f32(w); bias = _f32(bias)
    Cout, Cin, K = w.shape
    L = inp.shape[1]
    out = np.empty((Cout, L), np.float32)
    lib().aria_cuda_conv1d(_p(out), _p(inp), _p(w), _p(bias), Cin, Cout, K, pad, L)
    return out


# ---- aria_hip.h host-pointer forms ----

def layernorm(x, gamma, beta, eps):
    x = _f32(x); gamma = _f32(gamma); beta = _f32(beta)
    dim = x.shape[-1]
    y = np.empty_like(x)
    check(lib().aria_hip_layernorm(_p(y), _p(x), _p(gamma), _p(beta), x.size // dim, dim, eps),
          "aria_hip_layernorm")
    return y


def rmsnorm_adaln(x, w, scale, shift, eps, rows_per_batch=0):
    x = _f32(x); w = _f32(w); scale = _f32(scale); shift = _f32(shift)
    dim = x.shape[-1]
    y = np.empty_like(x)
    check(lib().aria_hip_rmsnorm_adaln(_p(y), _p(x), _p(w), _p(scale), _p(shift), x.size // dim, dim,
                                       rows_per_batch, eps), "aria_hip_rmsnorm_adaln")
    return y


def ln_mod_gelu_res(x, gamma, beta, scale, shift, eps):
    """x [B, S, D], scale/shift [B, D]: gelu(LN(x)*(1+scale)+shift) + x, one pass."""
    x = _f32(x); gamma = _f32(gamma); beta = _f32(beta); scale = _f32(scale); shift = _f32(shift)
    B, S, D = x.shape
    out = np.empty_like(x)
    check(lib().aria_hip_ln_mod_gelu_res(_p(out), _p(x), _p(gamma), _p(beta), _p(scale), _p(shift),
                                         B * S, D, S, eps), "aria_hip_ln_mod_gelu_res")
    return out


def modulate(x, scale, shift, rows_per_batch=0):
    x = _f32(x); scale = _f32(scale); shift = _f32(shift)
    dim = x.shape[-1]
    y = np.empty_like(x)
    check(lib().aria_hip_modulate(_p(y), _p(x), _p(scale), _p(shift), x.size // dim, dim, rows_per_batch),
          "aria_hip_modulate")
    return y


def gate_residual(res, o, gate, bias=None, rows_per_batch=0):
    res = _f32(res); o = _f32(o); gate = _f32(gate); bias = _f32(bias)
    dim = res.shape[-1]
    out = np.empty_like(res)
    check(lib().aria_hip_gate_residual(_p(out), _p(res), _p(o), _p(gate), _p(bias), res.size // dim, dim,
                                       rows_per_batch), "aria_hip_gate_residual")
    return out


def glu_combine(proj, bias=None):
    proj = _f32(proj); bias = _f32(bias)
    inner = proj.shape[-1] // 2
    rows = proj.size // proj.shape[-1]
    out = np.empty(proj.shape[:-1] + (inner,), np.float32)
    check(lib().aria_hip_glu_combine(_p(out), _p(proj), _p(bias), rows, inner), "aria_hip_glu_combine")
    return out


def add(a, b):
    a = _f32(a); b = _f32(b)
    y = np.empty_like(a)
    check(lib().aria_hip_add(_p(y), _p(a), _p(b), a.size), "aria_hip_add")
    return y


def addto(y, a):
    """aria_addto (src/aria_ops.h:167): y += a, as aria_hip_add_dev with y aliasing its first input"""
    from .device import DeviceArray
    dy = DeviceArray.from_host(_f32(y)); da = DeviceArray.from_host(_f32(a))
    try:
        check(lib().aria_hip_add_dev(dy.p, dy.p, da.p, dy.nbytes // 4, None), "aria_hip_add_dev")
        check(lib().aria_hip_stream_sync(None), "aria_hip_add_dev")
        return dy.to_host()
    finally:
        dy.free(); da.free()


def scale(x, s):
    """aria_scale (src/aria_ops.h:168): y = x * s (returns y)"""
    from .device import DeviceArray
    dx = DeviceArray.from_host(_f32(x)); dy = DeviceArray(dx.shape)
    try:
        check(lib().aria_hip_scale_dev(dy.p, dx.p, s, dx.nbytes // 4, None), "aria_hip_scale_dev")
        check(lib().aria_hip_stream_sync(None), "aria_hip_scale_dev")
        return dy.to_host()
    finally:
        dx.free(); dy.free()


def axpy(y, x, s):
    """aria_axpy (src/aria_ops.h:169): y += s * x (returns the new y)"""
    from .device import DeviceArray
    dy = DeviceArray.from_host(_f32(y)); dx = DeviceArray.from_host(_f32(x))
    try:
        check(lib().aria_hip_axpy_dev(dy.p, dx.p, s, dy.nbytes // 4, None), "aria_hip_axpy_dev")
        check(lib().aria_hip_stream_sync(None), "aria_hip_axpy_dev")
        return dy.to_host()
    finally:
        dy.free(); dx.free()


def pingpong(x, v, noise, tc, tn):
    y = _f32(x).copy()
    v = _f32(v); noise = _f32(noise)
    check(lib().aria_hip_pingpong(_p(y), _p(v), _p(noise), tc, tn, y.size), "aria_hip_pingpong")
    return y


def q8_quant(W):
    W = _f32(W)
    N, K = W.shape
    q = np.empty((N, K), np.int8); s = np.empty(N, np.float32)
    check(lib().aria_hip_q8_quant(_p(q), _p(s), _p(W), N, K), "aria_hip_q8_quant")
    return q, s


def q4_quant(W):
    W = _f32(W)
    N, K = W.shape
    q = np.empty((N, (K + 1) // 2), np.uint8); s = np.empty((N, 2 * ((K + 31) // 32)), np.float32)
    check(lib().aria_hip_q4_quant(_p(q), _p(s), _p(W), N, K), "aria_hip_q4_quant")
    return q, s


def linear_q8(x, q, s, b=None):
    """aria_linear_q8 (src/aria_quant.h:45): y = x dequant(q, s)^T + b, on MFMA."""
    x = _f32(x); b = _f32(b)
    M, K = x.shape
    N = q.shape[0]
    y = np.empty((M, N), np.float32)
    check(lib().aria_hip_linear_q8(_p(y), _p(x), _p(np.ascontiguousarray(q)), _p(np.ascontiguousarray(s)),
                                   _p(b), M, K, N), "aria_hip_linear_q8")
    return y


def linear_q4(x, q, s, b=None):
    """aria_linear_q4 (src/aria_quant.h:65): y = x dequant(q, s)^T + b, on MFMA."""
    x = _f32(x); b = _f32(b)
    M, K = x.shape
    N = q.shape[0]
    y = np.empty((M, N), np.float32)
    check(lib().aria_hip_linear_q4(_p(y), _p(x), _p(np.ascontiguousarray(q)), _p(np.ascontiguousarray(s)),
                                   _p(b), M, K, N), "aria_hip_linear_q4")
    return y


def linear_q8a8(x, q, s, b=None):
    """aria_linear_q8a8 (src/aria_quant.h:50): per-row int8 activations, exact int32 dot
    products on the int8 MFMA, y = acc * sx[m] * s[n] + b (bit-identical to the reference)."""
    x = _f32(x); b = _f32(b)
    M, K = x.shape
    N = q.shape[0]
    y = np.empty((M, N), np.float32)
    check(lib().aria_hip_linear_q8a8(_p(y), _p(x), _p(np.ascontiguousarray(q)), _p(np.ascontiguousarray(s)),
                                     _p(b), M, K, N), "aria_hip_linear_q8a8")
    return y


def q8_dequant(q, s):
    N, K = q.shape
    W = np.empty((N, K), np.float32)
    check(lib().aria_hip_q8_dequant(_p(W), _p(q), _p(s), N, K), "aria_hip_q8_dequant")
    return W


def q4_dequant(q, s, K):
    N = q.shape[0]
    W = np.empty((N, K), np.float32)
    check(lib().aria_hip_q4_dequant(_p(W), _p(q), _p(s), N, K), "aria_hip_q4_dequant")
    return W


# ---- MXFP4 and cross attention over ragged states (include/aria_hip.h; no counterpart in the reference) ----

def mx4_quant(x):
    """x [rows, K] -> codes u8 [rows, 16 * ceil(K/32)] and scale bytes u8 [rows, ceil(K/32)]."""
    x = _f32(x)
    rows, K = x.shape
    nb = (K + 31) // 32
    q = np.empty((rows, 16 * nb), np.uint8); s = np.empty((rows, nb), np.uint8)
    check(lib().aria_hip_mx4_quant(_p(q), _p(s), _p(x), rows, K), "aria_hip_mx4_quant")
    return q, s


def _mx4(q, s, K):
    q = np.ascontiguousarray(q, np.uint8); s = np.ascontiguousarray(s, np.uint8)
    nb = (K + 31) // 32
    if q.ndim != 2 or q.shape[1] != 16 * nb or s.shape != (q.shape[0], nb):
        raise ValueError(f"MXFP4 rows of {K} values are codes [rows, {16 * nb}] and scales [rows, {nb}]: "
                         f"got {q.shape} and {s.shape}")
    return q, s


def _bias(b, rows):
    b = _f32(b)
    if b is not None and b.size != rows:
        raise ValueError(f"the bias holds one value per weight row, [{rows}]: got {b.shape}")
    return b


def mx4_dequant(q, s, K):
    q, s = _mx4(q, s, K)
    y = np.empty((q.shape[0], K), np.float32)
    check(lib().aria_hip_mx4_dequant(_p(y), _p(q), _p(s), q.shape[0], K), "aria_hip_mx4_dequant")
    return y


def linear_mx4(x, q, s, b=None):
    """y = Q(x) W^T + b: x [M, K] quantised to MXFP4 in the call, W packed [N rows]."""
    x = _f32(x)
    M, K = x.shape
    q, s = _mx4(q, s, K)
    b = _bias(b, q.shape[0])
    y = np.empty((M, q.shape[0]), np.float32)
    check(lib().aria_hip_linear_mx4(_p(y), _p(x), _p(q), _p(s), _p(b), M, K, q.shape[0]), "aria_hip_linear_mx4")
    return y


def glu_mx4(x, q, s, b=None):
    """v * silu(g) with [v | g] = Q(x) W^T + b, W packed [2 * inner rows]."""
    x = _f32(x)
    M, K = x.shape
    q, s = _mx4(q, s, K)
    b = _bias(b, q.shape[0])
    inner = q.shape[0] // 2
    if q.shape[0] != 2 * inner:
        raise ValueError("a gated projection has an even number of weight rows")
    y = np.empty((M, inner), np.float32)
    check(lib().aria_hip_glu_mx4(_p(y), _p(x), _p(q), _p(s), _p(b), M, K, inner), "aria_hip_glu_mx4")
    return y


def cross_attention(q, k, v, kv_len=None, mask=None):
    """q [B, H, Nq, D], k / v [B, Hkv, Nk, D] (rounded to fp16), kv_len [B], mask [B, Nk] (nonzero =
    attend) -> [B, Nq, H * D]; a row without a valid key is zero."""
    q = _f32(q); k = _f32(k); v = _f32(v)
    B, H, Nq, D = q.shape
    Hkv, Nk = k.shape[1:3]
    if k.shape != (B, Hkv, Nk, D) or v.shape != k.shape:
        raise ValueError(f"k and v are [{B}, Hkv, Nk, {D}]: got {k.shape} and {v.shape}")
    if kv_len is not None:
        kv_len = np.ascontiguousarray(np.clip(kv_len, 0, Nk), np.int32)   # in the type they come in: 2^32 is not 0
        if kv_len.shape != (B,):
            raise ValueError(f"kv_len holds one length per sequence: got {kv_len.shape}")
    if mask is not None:
        mask = np.ascontiguousarray(np.asarray(mask) != 0, np.uint8)
        if mask.shape != (B, Nk):
            raise ValueError(f"mask is [{B}, {Nk}]: got {mask.shape}")
    out = np.empty((B, Nq, H * D), np.float32)
    check(lib().aria_hip_cross_attention_f16(_p(out), _p(q), _p(k), _p(v), _p(kv_len), _p(mask), B, H, Hkv, Nq, Nk, D),
          "aria_hip_cross_attention_f16")
    return out


# ---- rotary positions by table, e4m3 rows, attention over shared prefixes (include/aria_hip.h; no counterpart in the
# reference) ----

SCALINGS = {"none": 0, "linear": 1, "base": 2, "turns": 3}


def _strides(desc, name, N, heads, D):
    """packed [B, N, heads, D]"""
    for axis, n in (("batch", N * heads * D), ("token", heads * D), ("head", D)):
        setattr(desc, f"{name}_{axis}", n)


class _Device:
    """The device arrays of one call."""

    def __enter__(self):
        self.held = []
        return self

    def __exit__(self, *exc):
        for a in self.held:
            a.free()

    def put(self, a, dtype=np.float32):
        from .device import DeviceArray
        if a is None:
            return None
        self.held.append(DeviceArray.from_host(np.ascontiguousarray(a, dtype)))
        return self.held[-1]

    def new(self, shape, dtype=np.float32):
        from .device import DeviceArray
        self.held.append(DeviceArray(shape, dtype))
        return self.held[-1]

    def cache(self, B, heads, slots, D):
        from .cache import Cache
        c = Cache(B, heads, slots, D)
        self.held.append(c)
        return c


def _d(a):
    return None if a is None else a.p


def _call(fn, *args):
    check(getattr(lib(), fn)(*args), fn)
    check(lib().aria_hip_stream_sync(None), fn)


def rotary_tables(n, rot, first=0, base=10000.0, scaling="none", factor=1.0, trained=1.0, low=0.0, high=1.0, gain=1.0):
    """cos, sin [n, rot/2] of positions first .. first + n - 1."""
    from . import RotaryScaling
    a = RotaryScaling(rot=rot, kind=SCALINGS[scaling], base=base, factor=factor, trained=trained, low=low, high=high, gain=gain)
    with _Device() as dev:
        c, s = (dev.new((max(n, 0), max(rot, 0) // 2)) for _ in range(2))
        _call("aria_hip_rotary_table_dev", c.p, s.p, a, first, n, None)
        return c.to_host(), s.to_host()


def _int32(x):
    """held to 32 bits, so that 2^32 does not become 0"""
    return None if x is None else np.clip(np.asarray(x), -2 ** 31, 2 ** 31 - 1)


def _positions(pos, first, B, N):
    if pos is not None and np.shape(pos) != (B, N):
        raise ValueError(f"pos holds a position for each token, [{B}, {N}]: got {np.shape(pos)}")
    if first is not None and np.shape(first) != (B,):
        raise ValueError(f"first holds a position for each sequence, [{B}]: got {np.shape(first)}")
    return _int32(pos), _int32(first)


def rotary(q, cos, sin, k=None, pos=None, first=None, interleaved=False, inverse=False):
    """q [B, N, H, D] (and k [B, N, Hk, D]) rotated by rows of cos, sin [npos, rot/2]; tokens whose position lies outside
    the tables come back as they are."""
    from . import Rotary
    q = _f32(q); k = _f32(k); cos = _f32(cos); sin = _f32(sin)
    B, N, H, D = q.shape
    if cos.shape != sin.shape or cos.ndim != 2:
        raise ValueError(f"cos and sin are [positions, rot / 2]: got {cos.shape} and {sin.shape}")
    if k is not None and (k.shape[:2] != (B, N) or k.shape[3] != D):
        raise ValueError(f"k is [{B}, {N}, heads, {D}]: got {k.shape}")
    pos, first = _positions(pos, first, B, N)
    with _Device() as dev:
        dq, dk = dev.put(q), dev.put(k)
        a = Rotary(q=dq.p, q_out=dq.p, k=_d(dk), k_out=_d(dk), cos=dev.put(cos).p, sin=dev.put(sin).p, pos=_d(dev.put(pos, np.int32)),
                   first=_d(dev.put(first, np.int32)), pos_stride=N, type=0, B=B, N=N, Hq=H, Hk=0 if k is None else k.shape[2], D=D,
                   rot=2 * cos.shape[1], npos=cos.shape[0], interleaved=interleaved, inverse=inverse)
        for n in ("q", "qo"):
            _strides(a, n, N, H, D)
        for n in ("k", "ko"):
            _strides(a, n, N, a.Hk, D)
        _call("aria_hip_rotary_dev", a, None)
        return dq.to_host() if k is None else (dq.to_host(), dk.to_host())


def _write(dev, c, k, v, N):
    from . import KVWrite
    a = KVWrite(cache=c.desc, k=k.p, v=v.p, type=0, N=N)
    for n in ("k", "v"):
        _strides(a, n, N, c.heads, c.D)
    _call("aria_hip_kv_write_dev", a, None)


def e4m3_rows(x):
    """x [..., D] as rows of the cache: codes u8 [..., D] and scale bytes u8 [...]."""
    x = _f32(x)
    D = x.shape[-1]
    n = x.size // D if D else 0
    with _Device() as dev:
        c, d = dev.cache(1, 1, n, D), dev.put(x)
        _write(dev, c, d, d, n)
        return c.codes[0].to_host().reshape(x.shape), c.scales[0].to_host().reshape(x.shape[:-1])


def e4m3_values(codes, scales):
    """The values of such rows, fp32."""
    from . import KVRead
    codes = np.ascontiguousarray(codes, np.uint8); scales = np.ascontiguousarray(scales, np.uint8)
    if scales.shape != codes.shape[:-1]:
        raise ValueError(f"one scale byte for each row of codes: got {codes.shape} and {scales.shape}")
    D, n = codes.shape[-1], scales.size
    with _Device() as dev:
        c, y = dev.cache(1, 1, n, D), dev.new((n, D))
        c.codes[0].upload(codes.reshape(1, 1, n, D))
        c.scales[0].upload(scales.reshape(1, 1, n))
        a = KVRead(cache=c.desc, k=y.p, type=0, N=n)
        _strides(a, "k", n, 1, D)
        _call("aria_hip_kv_read_dev", a, None)
        return y.to_host().reshape(codes.shape)


def prefix_attention(q, prefix_k, prefix_v, k=None, v=None, prefix_len=None, own_len=None, first=None, scale=None):
    """q [B, Nq, H, D] (rounded to fp16) over prefixes [P, n, Hkv, D] (sequence b reads prefix b // (B / P)) and own keys and values
    [B, m, Hkv, D], both cached as e4m3 rows in the call and held to fp16's range; first [B]: query t of sequence b sees own keys up to first[b] + t
    -> [B, Nq, H, D] fp32."""
    from . import PrefixAttention
    q = _f32(q)
    B, Nq, H, D = q.shape
    pk = _f32(prefix_k); pv = _f32(prefix_v)
    P, n, Hkv = pk.shape[:3]
    k = np.zeros((B, 0, Hkv, D), np.float32) if k is None else _f32(k)
    v = np.zeros((B, 0, Hkv, D), np.float32) if v is None else _f32(v)
    m = k.shape[1]
    if pk.shape != (P, n, Hkv, D) or pv.shape != pk.shape or k.shape != (B, m, Hkv, D) or v.shape != k.shape:
        raise ValueError(f"keys and values are [prefixes, n, heads, {D}] and [{B}, m, heads, {D}]: got {pk.shape}, {pv.shape}, "
                         f"{k.shape} and {v.shape}")
    lens = []
    for x, rows, cap in ((prefix_len, P, n), (own_len, B, m), (first, B, None)):
        if x is not None:
            x = np.asarray(x)
            if x.shape != (rows,):
                raise ValueError(f"a length (or a first slot) for each of {rows}: got {x.shape}")
            x = _int32(x) if cap is None else np.clip(x, 0, cap)   # before 32 bits
        lens.append(x)
    with _Device() as dev:
        cp, co = dev.cache(P, Hkv, n, D), dev.cache(B, Hkv, m, D)
        for c, a, b, N in ((cp, pk, pv, n), (co, k, v, m)):
            if N:
                _write(dev, c, dev.put(a), dev.put(b), N)
        dq, out = dev.put(q, np.float16), dev.new((B, Nq, H, D))
        a = PrefixAttention(q=dq.p, out=out.p, prefix=cp.desc, own=co.desc, type=1, out_f32=1, B=B, H=H, Nq=Nq,
                            scale=1.0 / np.sqrt(D) if scale is None else scale)
        a.prefix_len, a.own_len, a.first = (_d(dev.put(x, np.int32)) for x in lens)
        for s in ("q", "o"):
            _strides(a, s, Nq, H, D)
        ws = dev.new(max(1, lib().aria_hip_prefix_attention_ws_bytes(a)), np.uint8)
        _call("aria_hip_prefix_attention_dev", a, ws.p, None)
        return out.to_host()
