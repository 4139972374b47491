"""Rotary positions by table and the 8-bit cache through the C ABI, against their definitions in 64 bits
(oracle/states.py). Refusals run on the CPU."""
from __future__ import annotations

import numpy as np
import pytest

from conftest import randn, rng
from oracle import mx4, states

CODE = {"f32": 0, "f16": 1, "bf16": 2}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LARGEST = {"f32": 3.4028234663852886e38, "f16": 65504.0, "bf16": 3.3895313892515355e38}
LEAST = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}    # half a step of the smallest numbers


def cast(x, t):
    """x as the type's bits and as the values they hold"""
    x = np.asarray(x, np.float32)
    if t == "f32":
        return x, x
    if t == "f16":
        h = x.astype(np.float16)
        return h, h.astype(np.float32)
    u = mx4.bf16_bits(x)
    bad = ~np.isfinite(x)
    u = np.where(bad, (x.view(np.uint32) >> 16).astype(np.uint16) | np.where(np.isnan(x), 0x40, 0).astype(np.uint16), u)
    return u, mx4.bf16_value(u)


def back(a, t):
    return mx4.bf16_value(a) if t == "bf16" else a.astype(np.float32)


class Laid:
    """A tensor [B, N, heads, D] of a type on the device under some strides, in a buffer filled with 99 where it is not."""

    def __init__(self, a, layout="tokens", pad=0, offset=0):
        from aria_amd.device import DeviceArray as DA
        B, N, h, D = a.shape
        self.shape = a.shape
        if layout == "tokens":               # rows of a wider projection
            row = h * D + pad
            self.batch, self.token, self.head = N * row, row, D
        else:                                # heads first, rows of D + pad
            row = D + pad
            self.batch, self.token, self.head = h * N * row, row, N * row
        self.offset = offset
        self.host = np.full(B * max(self.batch, 1) + offset + 64, 99, a.dtype)
        self.view()[...] = a
        self.dev = DA.from_host(self.host)
        self.p = self.dev.p + offset * a.dtype.itemsize

    def view(self):
        s = self.host.itemsize
        B, N, h, D = self.shape
        return np.lib.stride_tricks.as_strided(self.host[self.offset:], self.shape, (self.batch * s, self.token * s, self.head * s, s))

    def get(self):
        """what the device holds, and whether anything beside the tensor changed"""
        before = self.host.copy()
        self.host = self.dev.to_host()
        got = self.view().copy()
        keep = self.host.copy()
        self.view()[...] = 0
        beside = self.host.copy()
        self.host = before
        self.view()[...] = 0
        same = np.array_equal(beside, self.host)
        self.host = keep
        return got, same


def strides(a, name, t):
    for axis in ("batch", "token", "head"):
        setattr(a, f"{name}_{axis}", getattr(t, axis))


def dev(x, dtype=np.int32):
    from aria_amd.device import DeviceArray as DA
    return None if x is None else DA.from_host(np.asarray(x, dtype))


def ptr(d):
    return None if d is None else d.p


# ---- CPU ----

P = 4096     # never dereferenced


def test_refusals_table():
    import aria_amd
    L = aria_amd.lib()

    def call(first=0, n=4, c=P, s=P, **kw):
        a = aria_amd.RotaryScaling(rot=64, kind=0, base=10000.0, factor=2.0, trained=4096.0, low=1.0, high=32.0, gain=1.0)
        for k, v in kw.items():
            setattr(a, k, v)
        return L.aria_hip_rotary_table_dev(c, s, a, first, n, None)
    nan, inf = float("nan"), float("inf")
    for kw in (dict(rot=0), dict(rot=63), dict(rot=258), dict(rot=-2), dict(kind=-1), dict(kind=4), dict(base=1.0), dict(base=nan),
               dict(base=inf), dict(gain=nan), dict(gain=inf), dict(kind=1, factor=0.0), dict(kind=1, factor=nan),
               dict(kind=2, rot=2), dict(kind=2, factor=-1.0), dict(kind=3, trained=0.0), dict(kind=3, low=2.0, high=2.0),
               dict(kind=3, low=nan), dict(kind=3, high=inf), dict(first=-1), dict(first=1 << 24, n=2), dict(n=-1), dict(c=None),
               dict(s=None), dict(c=P + 2), dict(kind=1, factor=1e-30), dict(first=1 << 40)):
        assert call(**kw) == -1, kw
        assert "invalid argument" in aria_amd.last_error()
    assert L.aria_hip_rotary_table_dev(P, P, None, 0, 1, None) == -1
    assert call(n=0, c=None, s=None) == 0


def test_refusal_of_a_far_first():
    """A first position near the end of 64 bits is refused, not added to."""
    import aria_amd
    L = aria_amd.lib()
    a = aria_amd.RotaryScaling(rot=64, kind=0, base=10000.0, factor=2.0, trained=4096.0, low=1.0, high=32.0, gain=1.0)
    for first in ((1 << 63) - 1, (1 << 63) - 4, -(1 << 63), (1 << 24) + 1):
        assert L.aria_hip_rotary_table_dev(P, P, a, first, 4, None) == -1
        assert "invalid argument" in aria_amd.last_error()


def test_refusals_rotary():
    import aria_amd
    L = aria_amd.lib()

    def call(**kw):
        a = aria_amd.Rotary(q=P, k=P, q_out=P, k_out=P, cos=P, sin=P, type=1, B=2, N=3, Hq=4, Hk=2, D=64, rot=32, npos=8)
        for k, v in kw.items():
            setattr(a, k, v)
        return L.aria_hip_rotary_dev(a, None)
    for kw in (dict(type=3), dict(type=-1), dict(B=-1), dict(N=-1), dict(B=1 << 20, N=1 << 11), dict(D=63), dict(D=0), dict(D=258),
               dict(rot=31), dict(rot=66), dict(rot=-2), dict(npos=-1), dict(Hq=-1), dict(Hk=1 << 17), dict(q_out=None), dict(k=None),
               dict(q=P + 1), dict(k_out=P + 1), dict(type=0, q=P + 2), dict(cos=P + 2), dict(pos=P + 1), dict(first=P + 2),
               dict(q_batch=-1), dict(ko_head=-8), dict(pos_stride=-1), dict(cos=None), dict(sin=None), dict(q=None, q_out=None)):
        assert call(**kw) == -1, kw
        assert "invalid argument" in aria_amd.last_error()
    assert L.aria_hip_rotary_dev(None, None) == -1
    assert call(B=0, cos=None) == 0 and call(N=0) == 0


def test_refusals_cache():
    import aria_amd
    L = aria_amd.lib()

    def call(**kw):
        c = aria_amd.KVCache(k=P, v=P, k_scale=P, v_scale=P, batch=4096, head=1024, token=64, s_batch=32, s_head=16, B=2, Hkv=2,
                             D=64, cap=16)
        w = aria_amd.KVWrite(k=P, v=P, cos=P, sin=P, type=1, N=3, rot=32, npos=8)
        r = aria_amd.KVRead(k=P, v=P, type=1, N=3)
        for n, v in kw.items():
            for a in (c, w, r):
                if hasattr(a, n) and not (a is not c and n in ("k", "v")):
                    setattr(a, n, v)
        w.cache = r.cache = c
        return L.aria_hip_kv_write_dev(w, None), L.aria_hip_kv_read_dev(r, None)
    for kw in (dict(D=8), dict(D=24), dict(D=272), dict(Hkv=0), dict(Hkv=1 << 17), dict(B=-1), dict(B=1 << 17), dict(cap=-1),
               dict(k=None), dict(v_scale=None), dict(k=P + 8), dict(v=P + 4), dict(token=72), dict(batch=-16), dict(s_head=-1),
               dict(type=3), dict(N=-1), dict(first=P + 1), dict(count=P + 2)):
        assert call(**kw) == (-1, -1), kw
    for kw in (dict(rot=33), dict(rot=66), dict(cos=None), dict(sin=P + 1), dict(npos=-1), dict(q=P), dict(Hq=2), dict(q_out=P),
               dict(pos=P + 2), dict(pos_stride=-1), dict(k_token=-1), dict(cos=None, sin=None)):
        assert call(**kw)[0] == -1, kw
    assert call(B=0)[0] == 0 and call(N=0) == (0, 0)
    assert L.aria_hip_kv_write_dev(None, None) == -1 and L.aria_hip_kv_read_dev(None, None) == -1


def test_oracle_rows():
    """Every code's value is its own, halves go to the even code, 448 is reached and never passed."""
    code, byte = states.rows(np.append(states.E4M3[::-1], 0.0)[None])
    assert byte[0] == 127 and (code[0, :127] == np.arange(126, -1, -1)).all()
    mid = np.concatenate(([448.0], states.MIDDLE))
    code, byte = states.rows(mid[None])
    assert byte[0] == 127 and (code[0, 1:] == [i + i % 2 for i in range(126)]).all()
    for top, want in ((448.0, 127), (448.5, 128), (1.75, 119), (1.7500001, 120), (2.0 ** -130, 1), (0.0, 1), (3.4e38, 247)):
        assert states.rows(np.array([[top, 0]]))[1][0] == want, top


# ---- GPU ----

@pytest.mark.gpu
@pytest.mark.parametrize("rot,first,n,kw", [
    (64, 0, 33, {}), (32, 1000, 17, {}), (2, 0, 5, {}), (6, 7, 1, {}), (128, (1 << 24) - 63, 64, {}), (256, 131000, 70, {}),
    (64, 0, 40, dict(kind=1, factor=4.0)), (64, 5, 40, dict(kind=2, factor=8.0)), (128, 100000, 40, dict(kind=3, factor=8.0,
     trained=16384.0, low=1.0, high=32.0)), (50, 3, 129, dict(kind=3, factor=2.5, trained=512.0, low=0.5, high=4.0, base=500000.0)),
    (64, 4096, 3, dict(gain=1.2079)), (4, 0, 9, dict(kind=2, factor=3.0))])
def test_table(hip, rot, first, n, kw):
    from aria_amd.device import DeviceArray as DA, sync
    print(f"[gpu] table rot {rot} first {first} n {n} {kw}", flush=True)
    d = [DA.from_host(np.full((n + 1) * (rot // 2), 99, np.float32)) for _ in range(2)]
    full = dict(kind=0, base=10000.0, factor=1.0, trained=1.0, low=0.0, high=1.0, gain=1.0) | kw
    hip.check(hip.lib().aria_hip_rotary_table_dev(d[0].p, d[1].p, hip.RotaryScaling(rot=rot, **full), first, n, None))
    sync()
    # the angle: turns p f / 2 pi with f / 2 pi and the product rounded to 53 bits (and pow to about one step more), 2 pi 2^-52 of
    # them each; what is left of a turn as an fp32 number of half turns (pi 2^-25), the functions (2^-22 a step and a half of
    # 1), the gain and the product with it (half a step each)
    turns = (first + n) * float(np.max(states.frequencies(rot, **{k: v for k, v in full.items() if k != "gain"}))) / (2 * np.pi)
    tol = full["gain"] * (2 * np.pi * turns * 4 * 2.0 ** -53 + np.pi * 2.0 ** -25 + 2.0 ** -22 + 2 * 2.0 ** -24)
    for got, want in zip(d, states.table(rot, first, n, **kw)):
        got = got.to_host().reshape(n + 1, -1)
        assert (got[n] == 99).all()
        assert np.abs(got[:n] - want).max() <= tol, np.abs(got[:n] - want).max()


def some_table(rot, npos):
    c, s = states.table(rot, 0, npos)
    return c.astype(np.float32), s.astype(np.float32)


def rotated(x, cos, sin, at, inter, inverse=False):
    """x [B, N, h, D] by the rows `at` [B, N] of the tables; rows outside stay; (values, products' magnitudes, rows inside)"""
    ok = (at >= 0) & (at < len(cos))
    i = np.where(ok, at, 0)
    y, mag = states.rotate(x, cos[i][:, :, None], sin[i][:, :, None], inter, inverse)
    return y, mag, ok


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("B,N,H,Hk,D,rot,layout,pad", [
    (1, 1, 1, 1, 2, 2, "tokens", 0), (2, 5, 4, 2, 64, 32, "heads", 0), (3, 33, 16, 4, 128, 128, "tokens", 8), (2, 17, 3, 0, 80, 74, "tokens", 3),
    (1, 9, 5, 5, 96, 48, "heads", 1), (5, 1, 8, 2, 128, 64, "tokens", 0), (2, 3, 2, 1, 256, 2, "tokens", 0), (1, 40, 2, 2, 256, 256, "heads", 0),
    (1, 4, 2, 1, 18, 10, "tokens", 0), (2, 6, 2, 2, 64, 0, "tokens", 0), (2, 300, 16, 4, 64, 64, "tokens", 0)])
def test_rotary(hip, t, inter, B, N, H, Hk, D, rot, layout, pad):
    from aria_amd.device import sync
    print(f"[gpu] rotary {t} {'pairs' if inter else 'halves'} B {B} N {N} H {H}/{Hk} D {D} rot {rot} {layout}", flush=True)
    r = rng(B * 1000 + N + D + rot)
    npos = 2 * N + 40
    cos, sin = some_table(rot, npos) if rot else (np.zeros((1, 0), np.float32),) * 2
    dc, ds = dev(np.append(cos.ravel(), 0), np.float32), dev(np.append(sin.ravel(), 0), np.float32)
    q, qv = cast(randn(r, (B, N, H, D)), t)
    k, kv = cast(randn(r, (B, N, max(Hk, 1), D)), t)
    for how in ("given", "first", "neither"):
        pos = r.integers(-2, npos + 2, (B, N + 3)) if how == "given" else None      # a few outside of the table: padding
        first = r.integers(0, npos - N, B) if how == "first" else None
        at = pos[:, :N] if how == "given" else (first[:, None] if how == "first" else 0) + np.arange(N)[None, :].repeat(B, 0)
        for inverse in (False, True):
            lq, lk = Laid(q, layout, pad), Laid(k, layout, pad)
            oq, ok_ = (Laid(np.full(x.shape, 77, x.dtype), "heads" if layout == "tokens" else "tokens", pad) for x in (q, k))
            dp, df = dev(pos), dev(first)
            a = hip.Rotary(q=lq.p, q_out=oq.p, cos=dc.p, sin=ds.p, pos=ptr(dp), first=ptr(df), pos_stride=N + 3, type=CODE[t], B=B, N=N,
                           Hq=H, Hk=Hk, D=D, rot=rot, npos=npos, interleaved=inter, inverse=inverse)
            strides(a, "q", lq)
            strides(a, "qo", oq)
            if Hk:
                a.k, a.k_out = lk.p, ok_.p
                strides(a, "k", lk)
                strides(a, "ko", ok_)
            hip.check(hip.lib().aria_hip_rotary_dev(a, None))
            sync()
            for x, o in ((qv, oq),) + (((kv, ok_),) if Hk else ()):
                want, mag, ok = rotated(x, cos, sin, at, inter, inverse)
                if rot == 0:
                    ok = np.ones((B, N), bool)
                got, beside = o.get()
                assert beside, "written beside the rows"
                assert (got[~ok] == 77).all(), "a padding token was written"
                # fp32: the exact value's nearest (64-bit products); else products and sum in fp32, then the type's rounding
                tol = HALF_STEP[t] * np.abs(want) * 1.001 + LEAST[t] + (2.0 ** -50 if t == "f32" else 2.0 ** -22) * mag
                assert (np.abs(back(got, t) - want) <= tol)[ok].all()
                assert np.array_equal(got[ok][..., rot:], cast(x, t)[0][ok][..., rot:]), "plain dims are copied"


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("D,rot", [(4, 4), (8, 8), (12, 4), (24, 8), (24, 16), (36, 20), (36, 32), (40, 40), (132, 128), (136, 96), (232, 16),
                                   (256, 256), (256, 0)])
def test_rotary_odd_chunks(hip, t, inter, D, rot):
    """Odd numbers of 16-byte chunks, one chunk, more lanes than chunks, and the widest rows."""
    test_rotary(hip, t, inter, 2, 9, 5, 3, D, rot, "tokens", 3)


@pytest.mark.gpu
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("D,rot", [(64, 32), (80, 74), (128, 128)])
def test_rotary_in_place_and_back(hip, inter, D, rot):
    """In place; the inverse is the adjoint: <R x, g> = <x, R' g>, and R' R x is x."""
    from aria_amd.device import sync
    r = rng(D + rot)
    B, N, H = 2, 21, 6
    cos, sin = some_table(rot, 64)
    dc, ds = dev(cos, np.float32), dev(sin, np.float32)
    x, g = randn(r, (B, N, H, D)), randn(r, (B, N, H, D))

    def run(lx, inverse):
        a = hip.Rotary(q=lx.p, q_out=lx.p, cos=dc.p, sin=ds.p, type=0, B=B, N=N, Hq=H, D=D, rot=rot, npos=64, interleaved=inter,
                       inverse=inverse)
        strides(a, "q", lx)
        strides(a, "qo", lx)
        hip.check(hip.lib().aria_hip_rotary_dev(a, None))
        sync()
        return lx.get()[0].astype(np.float64)
    lx = Laid(x)
    rx = run(lx, False)
    want, _, _ = rotated(x, cos, sin, np.arange(N)[None].repeat(B, 0), inter)
    assert np.abs(rx - want).max() <= 2.0 ** -24 * np.abs(want).max()
    rg = run(Laid(g), True)
    assert abs((rx * g).sum() - (x * rg).sum()) <= 4 * 2.0 ** -24 * (np.abs(rx * g).sum() + np.abs(x * rg).sum())
    # a difference: R is linear, so (R(x + g) - R x) = R g to the roundings of three results
    xg = run(Laid((x + g).astype(np.float32)), False)
    lg = run(Laid(g), False)
    assert np.abs(xg - rx - lg).max() <= 8 * 2.0 ** -24 * (np.abs(xg).max() + np.abs(rx).max() + np.abs(lg).max())
    # cos^2 + sin^2 of the tables' fp32 numbers is 1 to 2^-23
    assert np.abs(run(lx, True) - x).max() <= 4 * 2.0 ** -23 * np.abs(x).max() * 2


class Cache:
    """A cache on the device, every byte 0xA5 before; codes [B, h, cap, D] (or tokens before heads), scale bytes [B, h, cap]."""

    def __init__(self, hip, B, h, cap, D, tokens_first=False):
        from aria_amd.device import DeviceArray as DA
        self.tokens_first = tokens_first
        shape = (B, cap, h, D) if tokens_first else (B, h, cap, D)
        fill = np.full(int(np.prod(shape)) + 64, 0xA5, np.uint8)
        self.code = [DA.from_host(fill) for _ in range(2)]
        self.byte = [DA.from_host(np.full(B * h * cap + 16, 0xA5, np.uint8)) for _ in range(2)]
        self.dims = B, h, cap, D
        self.c = hip.KVCache(k=self.code[0].p, v=self.code[1].p, k_scale=self.byte[0].p, v_scale=self.byte[1].p, B=B, Hkv=h, D=D,
                             cap=cap, batch=h * cap * D, head=D if tokens_first else cap * D, token=h * D if tokens_first else D,
                             s_batch=h * cap, s_head=cap)

    def get(self, i):
        """codes [B, cap, h, D] and bytes [B, cap, h] of keys (0) or values (1)"""
        B, h, cap, D = self.dims
        code, byte = self.code[i].to_host(), self.byte[i].to_host()
        n = B * h * cap
        assert (code[n * D:] == 0xA5).all() and (byte[n:] == 0xA5).all(), "written behind the cache"
        code = code[:n * D].reshape((B, cap, h, D) if self.tokens_first else (B, h, cap, D))
        return code if self.tokens_first else code.transpose(0, 2, 1, 3), byte[:n].reshape(B, h, cap).transpose(0, 2, 1)

    def put(self, i, code, byte):
        """the reverse of get"""
        code = code if self.tokens_first else code.transpose(0, 2, 1, 3)
        self.code[i].upload(np.append(np.ascontiguousarray(code).ravel(), np.full(64, 0xA5, np.uint8)))
        self.byte[i].upload(np.append(np.ascontiguousarray(byte.transpose(0, 2, 1)).ravel(), np.full(16, 0xA5, np.uint8)))


def cached(x, t):
    """states whose rows differ in size by far, with rows of zeros, ties and tiny numbers"""
    x = x * np.exp2(np.arange(x.shape[1]) % 23 - 11)[None, :, None, None]
    x.reshape(-1, x.shape[-1])[::7] = 0
    x[..., 1] = np.sign(x[..., 1]) * np.abs(x).max(-1) * 0.53125          # a half between two codes where the largest is 1.75 2^e
    x[..., 0] = np.abs(x).max(-1)
    return cast(x.astype(np.float32), t)


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("B,N,h,D,rot,layout,pad,Hq", [
    (1, 1, 1, 16, 0, "tokens", 0, 0), (2, 5, 2, 64, 32, "heads", 0, 4), (3, 33, 4, 128, 128, "tokens", 8, 16), (2, 17, 3, 80, 74, "tokens", 3, 3),
    (4, 1, 2, 128, 64, "tokens", 0, 8), (2, 70, 1, 256, 256, "heads", 1, 0), (3, 9, 5, 96, 0, "tokens", 0, 5), (2, 300, 8, 64, 64, "tokens", 0, 0),
    (1, 12, 2, 256, 2, "tokens", 0, 1)])
def test_write_and_read(hip, t, inter, B, N, h, D, rot, layout, pad, Hq):
    from aria_amd.device import sync
    L = hip.lib()
    r = rng(B + N + D + rot)
    cap = N + 37
    cos, sin = some_table(rot, cap) if rot else (None, None)
    dc, ds = dev(cos, np.float32), dev(sin, np.float32)
    k, kv = cached(randn(r, (B, N, h, D)), t)
    v, vv = cached(randn(r, (B, N, h, D)), t)
    q, qv = cast(randn(r, (B, N, max(Hq, 1), D)), t)
    lk, lv, lq = Laid(k, layout, pad), Laid(v, "heads", 0), Laid(q, layout, pad)
    for case in ("plain", "ragged", "edges"):
        print(f"[gpu] write {t} {'pairs' if inter else 'halves'} B {B} N {N} h {h} D {D} rot {rot} {case}", flush=True)
        first = None if case == "plain" else r.integers(0, cap - N + 1, B)
        count = None if case == "plain" else r.integers(0, N + 2, B)
        if case == "edges":                  # slots before and behind the cache, counts below zero
            first = r.integers(-N, cap + 1, B)
            count = np.where(np.arange(B) % 3 == 1, -4, N + 5)
        pos = r.integers(-1, cap + 1, (B, N)) if case == "edges" and rot else None
        c = Cache(hip, B, h, cap, D, tokens_first=case == "ragged")
        oq = Laid(np.full(q.shape, 77, q.dtype))
        df, dn, dp = dev(first), dev(count), dev(pos)
        w = hip.KVWrite(cache=c.c, k=lk.p, v=lv.p, cos=ptr(dc), sin=ptr(ds), pos=ptr(dp), first=ptr(df), count=ptr(dn), pos_stride=N,
                        type=CODE[t], N=N, rot=rot, npos=cap, interleaved=inter)
        strides(w, "k", lk)
        strides(w, "v", lv)
        if Hq:
            w.q, w.q_out, w.Hq = lq.p, oq.p, Hq
            strides(w, "q", lq)
            strides(w, "qo", oq)
        hip.check(L.aria_hip_kv_write_dev(w, None))
        sync()
        slot = (np.zeros(B, int) if first is None else first)[:, None] + np.arange(N)
        at = slot if pos is None else pos
        told = np.arange(N)[None] < (np.full(B, N) if count is None else count)[:, None]
        if rot:
            rk, _, inside = rotated(kv, cos, sin, at, inter)
            told &= inside
        else:
            rk = kv
        fits = told & (slot >= 0) & (slot < cap)
        for i, x in ((0, rk.astype(np.float32)), (1, vv)):
            code, byte = np.full((B, cap, h, D), 0xA5, np.uint8), np.full((B, cap, h), 0xA5, np.uint8)
            wc, wb = states.rows(x)
            for b in range(B):
                code[b, slot[b][fits[b]]], byte[b, slot[b][fits[b]]] = wc[b][fits[b]], wb[b][fits[b]]
            gc, gb = c.get(i)
            assert np.array_equal(gb, byte), "bytes of " + "kv"[i]
            assert np.array_equal(gc, code), "codes of " + "kv"[i]
        if Hq:
            got, beside = oq.get()
            want, mag = (rotated(qv, cos, sin, at, inter)[:2] if rot else (qv.astype(np.float64), 0 * qv))
            tol = HALF_STEP[t] * np.abs(want) * 1.001 + LEAST[t] + (2.0 ** -50 if t == "f32" else 2.0 ** -22) * mag
            assert beside and (got[~told] == 77).all() and (np.abs(back(got, t) - want) <= tol)[told].all()
        # back, in every type
        for y in ("f32", "f16", "bf16"):
            ok_, ov = (Laid(np.full((B, N, h, D), 77, cast(np.zeros(1), y)[0].dtype), "heads" if n else "tokens", 8 * n) for n in (0, 1))
            a = hip.KVRead(cache=c.c, k=ok_.p, v=ov.p, first=ptr(df), count=ptr(dn), type=CODE[y], N=N)
            strides(a, "k", ok_)
            strides(a, "v", ov)
            hip.check(L.aria_hip_kv_read_dev(a, None))
            sync()
            here = (np.arange(N)[None] < (np.full(B, N) if count is None else count)[:, None]) & (slot >= 0) & (slot < cap)
            for i, o in ((0, ok_), (1, ov)):
                code, byte = c.get(i)
                s = np.where(here, slot, 0)
                want = states.values(code[np.arange(B)[:, None], s], byte[np.arange(B)[:, None], s])
                want = cast(np.clip(want, -LARGEST[y], LARGEST[y]).astype(np.float32), y)[1]     # held to the type's range
                got, beside = o.get()
                assert beside and (got[~here] == 77).all()
                assert np.array_equal(back(got, y)[here], want[here])


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_rows_that_are_not_finite(hip, t):
    """Such a row is NaN as a whole, its neighbours are not; the type's largest and smallest numbers."""
    from aria_amd.device import sync
    B, N, h, D = 1, 12, 2, 64
    x = randn(rng(3), (B, N, h, D))
    x[0, 2, 0, 5], x[0, 4, 1, 63], x[0, 5, 0, 0] = np.nan, np.inf, -np.inf
    big = {"f32": 3.4028234e38, "f16": 65504.0, "bf16": 3.3895314e38}[t]
    x[0, 7, 0], x[0, 8, 1] = 0, 0
    x[0, 7, 0, 3], x[0, 7, 0, 4] = big, -big
    x[0, 8, 1, 9] = {"f32": 1e-45, "f16": 6e-8, "bf16": 1e-40}[t]
    x[0, 9] = -0.0
    k, kv = cast(x, t)
    lk = Laid(k)
    c = Cache(hip, B, h, N, D)
    w = hip.KVWrite(cache=c.c, k=lk.p, v=lk.p, type=CODE[t], N=N)
    strides(w, "k", lk)
    strides(w, "v", lk)
    hip.check(hip.lib().aria_hip_kv_write_dev(w, None))
    sync()
    code, byte = states.rows(kv)
    assert (byte == 255).sum() == 3
    for i in range(2):
        gc, gb = c.get(i)
        assert np.array_equal(gb, byte) and np.array_equal(gc, code)
    o = Laid(np.zeros((B, N, h, D), np.float32))
    a = hip.KVRead(cache=c.c, v=o.p, type=0, N=N)
    strides(a, "v", o)
    hip.check(hip.lib().aria_hip_kv_read_dev(a, None))
    sync()
    got = o.get()[0]
    assert np.array_equal(np.isnan(got).all(-1), byte == 255) and np.isfinite(got[byte != 255]).all()


@pytest.mark.gpu
def test_broadcast_states(hip):
    """Strides of zero on inputs: one row for all heads and tokens."""
    from aria_amd.device import sync
    B, N, h, D = 2, 6, 3, 64
    x, xv = cast(randn(rng(4), (1, 1, 1, D)), "f16")
    lx = Laid(x)
    c = Cache(hip, B, h, N, D)
    w = hip.KVWrite(cache=c.c, k=lx.p, v=lx.p, type=1, N=N)
    hip.check(hip.lib().aria_hip_kv_write_dev(w, None))
    sync()
    code, byte = states.rows(np.broadcast_to(xv, (B, N, h, D)))
    gc, gb = c.get(0)
    assert np.array_equal(gc, code) and np.array_equal(gb, byte)


@pytest.mark.gpu
def test_more_tokens_than_workgroups(hip):
    """Five million tokens of one pair each: workgroups take several shares."""
    from aria_amd.device import DeviceArray as DA, sync
    N = 5_000_003
    cos, sin = some_table(2, 64)
    x = randn(rng(8), (N, 2))
    pos = (np.arange(N, dtype=np.int64) * 7 % 64).astype(np.int32)
    dx, dy, dp, dc, ds = DA.from_host(x), DA((N, 2)), DA.from_host(pos), DA.from_host(cos), DA.from_host(sin)
    a = hip.Rotary(q=dx.p, q_out=dy.p, cos=dc.p, sin=ds.p, pos=dp.p, type=0, B=1, N=N, Hq=1, D=2, rot=2, npos=64, q_token=2, qo_token=2)
    hip.check(hip.lib().aria_hip_rotary_dev(a, None))
    sync()
    want, _ = states.rotate(x, cos[pos], sin[pos], False)
    assert np.abs(dy.to_host() - want).max() <= 2.0 ** -24 * np.abs(want).max()
