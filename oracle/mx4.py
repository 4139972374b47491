"""TEST INFRASTRUCTURE ONLY: MXFP4 and ragged cross attention from their definitions, numpy in 64 bits.

MXFP4: blocks of 32 along K share 2^(byte - 127); codes are sign and magnitude out of MAG. The
block exponent is floor(log2 max|x|) - 2, at least -127; a block that is not finite has byte 255.
"""
from __future__ import annotations

import numpy as np

MAG = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def bf16_bits(x):
    """fp32 -> bf16, to nearest even (finite values)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def bf16_value(u):
    return (np.ascontiguousarray(u, np.uint16).astype(np.uint32) << 16).view(np.float32)


def quant(x):
    """x [rows, K] -> codes u8 [rows, 16 nb], scale bytes u8 [rows, nb]."""
    x = np.asarray(x, np.float64)
    rows, K = x.shape
    nb = (K + 31) // 32
    b = np.zeros((rows, nb * 32))
    b[:, :K] = x
    b = b.reshape(rows, nb, 32)
    bad = ~np.isfinite(b).all(-1)
    a = np.where(bad[..., None], 0.0, np.abs(b))
    top = a.max(-1)
    e = np.where(top > 0, np.frexp(top)[1] - 1 - 2, -127)
    e = np.maximum(e, -127)
    v = np.ldexp(a, -e[..., None])
    code = np.zeros(v.shape, np.int64)
    for c in range(7):                       # a tie between codes c and c + 1 goes to the even one
        mid = (MAG[c] + MAG[c + 1]) / 2
        code += (v > mid) | ((v == mid) & ((c + 1) % 2 == 0))
    code |= np.where(bad[..., None], 0, np.signbit(b) * 8)
    code[np.broadcast_to(np.arange(32)[None, None] + 32 * np.arange(nb)[None, :, None] >= K, code.shape)] = 0
    q = (code[..., 0::2] | code[..., 1::2] << 4).astype(np.uint8).reshape(rows, 16 * nb)
    return q, np.where(bad, 255, e + 127).astype(np.uint8)


def dequant(q, s, K):
    """The values in 64 bits."""
    c = np.stack((q & 15, q >> 4), -1).reshape(q.shape[0], -1)
    v = np.where(c & 8, -1.0, 1.0) * MAG[c & 7]
    p = np.where(s == 255, np.nan, np.ldexp(1.0, s.astype(np.int64) - 127))
    return (v * np.repeat(p, 32, 1))[:, :K]


def linear(x, q, s, b=None):
    """(y, sum of |terms|) of Q(x) W^T + b for x [M, K] as given."""
    K = x.shape[1]
    xv, wv = dequant(*quant(x), K), dequant(q, s, K)
    y, t = xv @ wv.T, np.abs(xv) @ np.abs(wv).T
    return (y, t) if b is None else (y + b, t + np.abs(b))


def cross_attention(q, k, v, kv_len=None, mask=None, scale=None):
    """q [B, H, Nq, D], k / v [B, Hkv, Nk, D] -> (out [B, Nq, H, D], sum of p |v| of the same shape)."""
    B, H, Nq, D = q.shape
    Hkv, Nk = k.shape[1:3]
    scale = 1 / np.sqrt(D) if scale is None else scale
    out = np.zeros((B, Nq, H, D)); mag = np.zeros((B, Nq, H, D))
    for b in range(B):
        ok = np.ones(Nk, bool) if mask is None else mask[b] != 0
        if kv_len is not None:
            ok = ok & (np.arange(Nk) < kv_len[b])
        if not ok.any():
            continue
        for h in range(H):
            kk, vv = (t[b, h // (H // Hkv)][ok].astype(np.float64) for t in (k, v))
            sc = q[b, h].astype(np.float64) @ kk.T * scale
            p = np.exp(sc - sc.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            out[b, :, h], mag[b, :, h] = p @ vv, p @ np.abs(vv)
    return out, mag
