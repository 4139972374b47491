"""TEST INFRASTRUCTURE ONLY: rotary positions, e4m3 rows of keys and values, and attention over shared prefixes
from their definitions, numpy in 64 bits.
"""
from __future__ import annotations

import numpy as np

# the values of codes 0 .. 126 (127 is NaN)
E4M3 = np.array([(m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127])
MIDDLE = (E4M3[1:] + E4M3[:-1]) / 2


def frequencies(rot, kind=0, base=10000.0, factor=1.0, trained=1.0, low=0.0, high=1.0):
    """Radians a position of every pair (the kinds of aria_hip_rotary_scaling)."""
    i = np.arange(rot // 2, dtype=np.longdouble)
    base = np.longdouble(base)
    if kind == 2:
        base = base * np.longdouble(factor) ** (np.longdouble(rot) / (rot - 2))
    f = base ** (-2 * i / rot)
    if kind == 1:
        f = f / factor
    if kind == 3:
        w = np.clip((trained * f / (2 * np.pi) - low) / (high - low), 0, 1)
        f = f * (w + (1 - w) / factor)
    return f


def table(rot, first, n, gain=1.0, **kw):
    """cos, sin [n, rot/2] in 64 bits, the angles in more."""
    a = np.arange(first, first + n).astype(np.longdouble)[:, None] * frequencies(rot, **kw)
    return (np.cos(a) * gain).astype(np.float64), (np.sin(a) * gain).astype(np.float64)


def rotate(x, cos, sin, interleaved, inverse=False):
    """x [..., D] by cos, sin [..., rot/2] (the leading axes broadcast); also the sum of the products' magnitudes."""
    x, c, s = (np.asarray(a, np.float64) for a in (x, cos, sin))
    if inverse:
        s = -s
    h = c.shape[-1]
    ia, ib = (np.arange(h) * 2, np.arange(h) * 2 + 1) if interleaved else (np.arange(h), np.arange(h) + h)
    y, mag = x.copy(), np.zeros(x.shape)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia], mag[..., ib] = np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s)
    return y, mag


def rows(x):
    """x [..., D] (fp32 values) -> codes u8 [..., D], bytes u8 [...]."""
    x = np.asarray(x, np.float64)
    bad = ~np.isfinite(x).all(-1)
    a = np.where(bad[..., None], 0.0, np.abs(x))
    top = a.max(-1)
    byte = np.ones(top.shape, np.int64)
    for n in range(2, 255):                  # the smallest that brings the largest to 448 or less
        byte += top > np.ldexp(448.0, n - 1 - 127)
    v = np.ldexp(a, 127 - byte[..., None])
    code = np.searchsorted(MIDDLE, v, side="left")          # middles below v
    tie = (code < 126) & (MIDDLE[np.minimum(code, 125)] == v) & (code % 2 == 1)
    code = (code + tie) | (np.signbit(x).astype(np.int64) << 7)
    code = np.where(bad[..., None], 0x7F, code).astype(np.uint8)
    return code, np.where(bad, 255, byte).astype(np.uint8)


def values(code, byte):
    c = np.asarray(code).astype(np.int64)
    v = np.append(E4M3, np.nan)[c & 127] * np.where(c & 128, -1.0, 1.0)
    with np.errstate(invalid="ignore"):
        return np.where((np.asarray(byte) == 255)[..., None], np.nan, np.ldexp(v, np.asarray(byte).astype(np.int64)[..., None] - 127))


def attention(q, prefix, own, prefix_len=None, own_len=None, first=None, scale=None):
    """q [B, H, Nq, D]; prefix (k, v) [P, Hkv, n, D], own (k, v) [B, Hkv, m, D] -> out [B, Nq, H, D] and sum_j p_j |v_j|."""
    q = np.asarray(q, np.float64)
    B, H, Nq, D = q.shape
    P, Hkv, n = prefix[0].shape[:3]
    m = own[0].shape[2]
    scale = 1 / np.sqrt(D) if scale is None else scale
    out, mag = np.zeros((B, Nq, H, D)), np.zeros((B, Nq, H, D))
    for b in range(B):
        p = b // (B // P)
        ln = n if prefix_len is None else min(max(int(prefix_len[p]), 0), n)
        lm = m if own_len is None else min(max(int(own_len[b]), 0), m)
        for h in range(H):
            hk = h // (H // Hkv)
            k = np.concatenate((prefix[0][p, hk, :ln], own[0][b, hk, :lm])).astype(np.float64)
            v = np.concatenate((prefix[1][p, hk, :ln], own[1][b, hk, :lm])).astype(np.float64)
            for t in range(Nq):
                see = np.ones(ln + lm, bool)
                if first is not None:
                    see[ln:] = np.arange(lm) <= int(first[b]) + t
                if not see.any():
                    continue
                s = k[see] @ q[b, h, t] * scale
                w = np.exp(s - s.max())
                w = w / w.sum()
                out[b, t, h] = w @ v[see]
                mag[b, t, h] = w @ np.abs(v[see])
    return out, mag
