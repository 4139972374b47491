"""Cross attention over ragged encoder states through the C ABI, against the definition in 64 bits
(oracle/mx4.py). Refusals run on the CPU."""
from __future__ import annotations

import numpy as np
import pytest

from conftest import randn, rng
from oracle import mx4

CODE = {"f16": 1, "bf16": 2}
HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}


def cast(x, t):
    if t == "f16":
        h = x.astype(np.float16)
        return h, h.astype(np.float32)
    u = mx4.bf16_bits(x)
    return u, mx4.bf16_value(u)


def describe(hip, t, B, H, Hkv, Nq, Nk, D, scale=None):
    """The call's description with packed head-major q, k, v and a merged-head output."""
    return hip.CrossAttention(type=CODE[t], B=B, H=H, Hkv=Hkv, Nq=Nq, Nk=Nk, D=D,
                              scale=1 / np.sqrt(D) if scale is None else scale,
                              q_batch=H * Nq * D, q_head=Nq * D, q_token=D, k_batch=Hkv * Nk * D, k_head=Nk * D, k_token=D,
                              v_batch=Hkv * Nk * D, v_head=Nk * D, v_token=D, o_batch=Nq * H * D, o_head=D, o_token=H * D,
                              mask_stride=Nk)


# ---- CPU ----

def test_refusals():
    import aria_amd
    L = aria_amd.lib()
    p = 4096   # never dereferenced

    def call(ws=p, **kw):
        a = describe(aria_amd, "f16", 2, 4, 2, 3, 5, 64)
        a.q = a.k = a.v = a.out = p
        for n, v in kw.items():
            setattr(a, n, v)
        return L.aria_hip_cross_attention_dev(a, ws, None), L.aria_hip_cross_attention_ws_bytes(a)

    for kw in (dict(type=0), dict(type=3), dict(D=4), dict(D=12), dict(D=136), dict(D=0), dict(H=3), dict(Hkv=0), dict(H=0),
               dict(Nq=-1), dict(Nk=-1), dict(B=-1), dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(q=p + 2),
               dict(out=p + 8), dict(kv_len=p + 2), dict(k_token=60), dict(v_batch=-8), dict(o_token=12), dict(q_head=4),
               dict(Nq=1 << 30), dict(mask=p, mask_stride=-1), dict(scale=0.0), dict(scale=-0.1), dict(scale=float("nan")),
               dict(scale=float("inf"))):
        rc, ws = call(**kw)
        assert rc == -1 and ws == 0, kw
        assert "invalid argument" in aria_amd.last_error()
    assert call(ws=p + 8)[0] == -1
    assert L.aria_hip_cross_attention_dev(None, None, None) == -1 and L.aria_hip_cross_attention_ws_bytes(None) == 0
    assert call(B=0, q=None)[0] == 0 and call(Nq=0, out=None)[0] == 0     # nothing to do
    from aria_amd import ops
    z = np.zeros((2, 4, 3, 64), np.float32)
    with pytest.raises(ValueError):
        ops.cross_attention(z, z[:, :2], z[:, :3])
    with pytest.raises(ValueError):
        ops.cross_attention(z, z[:, :2], z[:, :2], kv_len=[1])
    with pytest.raises(ValueError):
        ops.cross_attention(z, z[:, :2], z[:, :2], mask=np.ones((2, 4)))
    with pytest.raises(aria_amd.HipError):
        ops.cross_attention(z[..., :12], z[:, :2, :, :12], z[:, :2, :, :12])


# ---- GPU ----

def tolerance(want, mag, q, k, v, t, out, scale, Nk):
    """fp32 scores: |ds| <= D 2^-23 sum |q||k| scale, and the exponent's rounding: |s| log2(e) 2^-23, both
    relative errors of p; p and the sum of p are the same rounded numbers (half a step each, and exp's
    own two); probabilities that fall under the type's smallest number against a row maximum of at
    least 1 cost 2^-24 each; then the output's rounding."""
    D = q.shape[-1]
    s = np.abs(q).max(initial=0) * np.abs(k[np.isfinite(k)]).max(initial=0) * D * scale
    d = (D + 4) * 2.0 ** -23 * s
    rel = 2 * (HALF_STEP[t] + d + 2.0 ** -21)
    vmax = np.abs(v[np.isfinite(v)]).max(initial=0)
    return rel * (mag + np.abs(want)) + Nk * 2.0 ** -24 * vmax + HALF_STEP[out] * np.abs(want) * 1.001 + 2.0 ** -25


def run(hip, t, q, k, v, kv_len=None, mask=None, out="same", layout="heads", scale=None, stream=None):
    """q [B, H, Nq, D], k / v [B, Hkv, Nk, D] already in the type; (result [B, Nq, H, D])."""
    from aria_amd.device import DeviceArray as DA, sync
    L = hip.lib()
    B, H, Nq, D = q.shape
    Hkv, Nk = k.shape[1:3]
    a = describe(hip, t, B, H, Hkv, Nq, Nk, D, scale)
    if layout == "heads":
        dq, dk, dv = (DA.from_host(x) if x.size else DA((8,), np.uint16) for x in (q, k, v))
        a.q, a.k, a.v = dq.p, dk.p, dv.p
    else:          # tokens first, k and v as one fused projection [B, Nk, 2, Hkv, D] inside wider rows
        dq = DA.from_host(np.ascontiguousarray(q.transpose(0, 2, 1, 3)))
        pad = 24
        kv = np.full((B, Nk, 2 * Hkv * D + pad), cast(np.array([np.nan], np.float32), t)[0][0], q.dtype)
        kv[:, :, :Hkv * D] = k.transpose(0, 2, 1, 3).reshape(B, Nk, -1)
        kv[:, :, Hkv * D:2 * Hkv * D] = v.transpose(0, 2, 1, 3).reshape(B, Nk, -1)
        dk = dv = DA.from_host(kv)
        row = 2 * Hkv * D + pad
        a.q, a.k, a.v = dq.p, dk.p, dk.p + Hkv * D * 2
        a.q_batch, a.q_head, a.q_token = Nq * H * D, D, H * D
        a.k_batch = a.v_batch = Nk * row
        a.k_head = a.v_head = D
        a.k_token = a.v_token = row
    guard = 2      # rows behind the last one
    ot = np.float32 if out == "f32" else q.dtype
    fill = np.full((B * Nq + guard, H * D), 99, ot)
    do = DA.from_host(fill)
    a.out, a.out_f32 = do.p, int(out == "f32")
    dl = DA.from_host(np.asarray(kv_len, np.int32)) if kv_len is not None else None
    dm = DA.from_host(np.asarray(mask, np.uint8)) if mask is not None and Nk else None
    a.kv_len, a.mask = dl.p if dl else None, dm.p if dm else None
    ws = DA(max(1, L.aria_hip_cross_attention_ws_bytes(a)), np.uint8)
    ws.upload(np.full(ws.shape, 0xFF, np.uint8))
    hip.check(L.aria_hip_cross_attention_dev(a, ws.p, stream))
    sync(stream)
    o = do.to_host()
    assert (o[B * Nq:] == 99).all(), "rows behind the last one were written"
    o = o[:B * Nq].reshape(B, Nq, H, D)
    return mx4.bf16_value(o) if o.dtype == np.uint16 else o.astype(np.float32)


def check(hip, t, B, H, Hkv, Nq, Nk, D, seed, kv_len=None, mask=None, out="same", layout="heads", spread=1.0):
    r = rng(seed)
    q, qv = cast(randn(r, (B, H, Nq, D)) * spread, t)
    k, kv = cast(randn(r, (B, Hkv, Nk, D)), t)
    v, vv = cast(randn(r, (B, Hkv, Nk, D)), t)
    print(f"[gpu] cross attention {t} B {B} H {H}/{Hkv} Nq {Nq} Nk {Nk} D {D} {layout}", flush=True)
    got = run(hip, t, q, k, v, kv_len, mask, out, layout)
    want, mag = mx4.cross_attention(qv, kv, vv, kv_len, mask)
    tol = tolerance(want, mag, qv, kv, vv, t, out if out == "f32" else t, 1 / np.sqrt(D), Nk)
    assert (np.abs(got - want) <= tol).all(), np.abs(got - want).max()
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("B,H,Hkv,Nq,Nk,D", [(1, 1, 1, 1, 1, 64), (2, 4, 2, 1, 33, 64), (1, 2, 2, 5, 64, 128), (3, 2, 1, 33, 65, 72),
                                             (1, 3, 3, 130, 257, 64), (2, 4, 1, 64, 100, 40), (1, 2, 2, 31, 700, 96),
                                             (1, 8, 1, 3, 1000, 128), (2, 1, 1, 257, 129, 8), (1, 6, 2, 50, 2111, 64),
                                             (1, 2, 1, 300, 520, 128)])
def test_full(hip, t, B, H, Hkv, Nq, Nk, D):
    check(hip, t, B, H, Hkv, Nq, Nk, D, seed=Nq + Nk + D)
    check(hip, t, B, H, Hkv, Nq, Nk, D, seed=Nq + Nk + D + 1, layout="tokens", out="f32", spread=3.0)


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("B,H,Hkv,Nq,Nk,D", [(2, 4, 4, 2000, 130, 64), (1, 16, 8, 1100, 600, 64), (3, 16, 16, 1000, 300, 64),
                                             (2, 8, 8, 1025, 1090, 128), (3, 16, 16, 1000, 200, 72), (8, 16, 16, 2050, 100, 64),
                                             (1, 8, 2, 700, 1100, 128)])
def test_many_rows(hip, t, B, H, Hkv, Nq, Nk, D):
    """Enough rows for every form of workgroup: two slices of the keys, one, and eight waves; ragged and masked."""
    check(hip, t, B, H, Hkv, Nq, Nk, D, seed=Nq + Nk)
    lens = [Nk - 1, Nk // 3, 0, Nk, 1, 64, 65, 70][:B]
    mask = (rng(Nq).random((B, Nk)) < 0.6).astype(np.uint8)
    check(hip, t, B, H, Hkv, Nq, Nk, D, seed=Nq, kv_len=lens, mask=mask, layout="tokens")


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("Nq,Nk,D", [(1, 200, 64), (40, 200, 128), (150, 500, 64), (3, 3000, 128)])
def test_lengths_and_masks(hip, t, Nq, Nk, D):
    """Every length from none over one tile's corners to all; a mask beside it; all masked away."""
    lens = [0, 1, 63, 64, 65, Nk - 1, Nk, Nk + 7, -3]      # as the description says: clamped to 0..Nk
    B = len(lens)
    r = rng(Nq + Nk)
    mask = (r.random((B, Nk)) < 0.5).astype(np.uint8) * 3
    mask[1], mask[2] = 0, 1
    mask[5, :130] = 0                                      # whole tiles masked
    got = check(hip, t, B, 4, 2, Nq, Nk, D, 11, kv_len=lens)
    assert (got[0] == 0).all() and (got[8] == 0).all()
    got = check(hip, t, B, 4, 2, Nq, Nk, D, 12, kv_len=lens, mask=mask, layout="tokens")
    assert (got[0] == 0).all() and (got[1] == 0).all()
    check(hip, t, B, 4, 2, Nq, Nk, D, 13, mask=mask)


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 72, 128])
def test_few_rows_many_tiles(hip, t, D):
    """Several tiles to each wave and split: lengths that end anywhere, with a mask and without, whole tiles of it gone."""
    B, Nk = 24, 2500
    r = rng(D)
    lens = [int(n) for n in r.integers(0, Nk + 1, B)]
    mask = (r.random((B, Nk)) < 0.8).astype(np.uint8)
    mask[3, 256:900] = 0
    mask[4, :2000] = 0
    check(hip, t, B, 8, 4, 2, Nk, D, seed=D, kv_len=lens)
    check(hip, t, B, 8, 4, 2, Nk, D, seed=D + 1, kv_len=lens, mask=mask, layout="tokens")
    check(hip, t, B, 8, 4, 2, Nk, D, seed=D + 2, mask=mask, spread=3.0)


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("Nq", [1, 70])
def test_anything_in_masked_places(hip, t, Nq):
    """NaN and Inf in masked keys and values, and behind the lengths, change no bit of the result."""
    r = rng(5)
    B, H, Hkv, Nk, D = 3, 4, 2, 190, 64
    q = cast(randn(r, (B, H, Nq, D)), t)[0]
    kf, vf = randn(r, (B, Hkv, Nk, D)), randn(r, (B, Hkv, Nk, D))
    lens = [190, 100, 0]
    mask = (r.random((B, Nk)) < 0.7).astype(np.uint8)
    gone = (mask == 0) | (np.arange(Nk)[None] >= np.array(lens)[:, None])
    want = run(hip, t, q, cast(kf, t)[0], cast(vf, t)[0], lens, mask)
    for bad in (np.nan, np.inf, -np.inf, 65504.0):
        k2, v2 = kf.copy(), vf.copy()
        k2[np.broadcast_to(gone[:, None, :], (B, Hkv, Nk))] = bad
        v2[np.broadcast_to(gone[:, None, :], (B, Hkv, Nk))] = bad
        got = run(hip, t, q, cast(k2, t)[0], cast(v2, t)[0], lens, mask)
        assert np.array_equal(got, want), bad


@pytest.mark.gpu
@pytest.mark.parametrize("Nq", [1, 40])
def test_no_keys(hip, Nq):
    """An encoder without states: zeros, with neither k nor v."""
    from aria_amd.device import DeviceArray as DA, sync
    a = describe(hip, "f16", 2, 4, 2, Nq, 0, 64)
    dq, do = DA.from_host(np.ones((2, 4, Nq, 64), np.float16)), DA.from_host(np.ones((2, Nq, 256), np.float16))
    a.q, a.out = dq.p, do.p
    hip.check(hip.lib().aria_hip_cross_attention_dev(a, None, None))
    sync()
    assert (do.to_host() == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("Nq,Nk", [(1, 400), (90, 400)])
def test_peaked_scores(hip, t, Nq, Nk):
    """Scores far apart, rising and falling along the keys: the running maximum moves at every tile."""
    r = rng(9)
    D = 64
    q = np.ones((1, 2, Nq, D), np.float32)
    ramp = np.linspace(-12, 12, Nk)[None, None, :, None] / 8
    k = np.concatenate([ramp, -ramp], 1) * np.ones((1, 2, Nk, D))
    v = randn(r, (1, 2, Nk, D))
    (q, qv), (k, kv), (v, vv) = cast(q, t), cast(k.astype(np.float32), t), cast(v, t)
    got = run(hip, t, q, k, v)
    want, mag = mx4.cross_attention(qv, kv, vv)
    assert (np.abs(got - want) <= tolerance(want, mag, qv, kv, vv, t, t, 1 / 8, Nk)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("Nq", [1, 50])
def test_broadcast_states(hip, Nq):
    """One prompt's states for every sequence: batch strides of zero; equal to the copied states' bits."""
    from aria_amd.device import DeviceArray as DA, sync
    r = rng(21)
    B, H, Nk, D = 3, 4, 150, 64
    q = randn(r, (B, H, Nq, D)).astype(np.float16)
    k, v = (randn(r, (1, H, Nk, D)).astype(np.float16) for _ in range(2))
    want = run(hip, "f16", q, np.repeat(k, B, 0), np.repeat(v, B, 0), [150, 20, 97])
    a = describe(hip, "f16", B, H, H, Nq, Nk, D)
    d = [DA.from_host(x) for x in (q, k, v)]
    do, dl = DA((B, Nq, H * D), np.float16), DA.from_host(np.array([150, 20, 97], np.int32))
    a.q, a.k, a.v, a.out, a.kv_len = d[0].p, d[1].p, d[2].p, do.p, dl.p
    a.k_batch = a.v_batch = 0
    ws = DA(max(1, hip.lib().aria_hip_cross_attention_ws_bytes(a)), np.uint8)
    hip.check(hip.lib().aria_hip_cross_attention_dev(a, ws.p, None))
    sync()
    assert np.array_equal(do.to_host().reshape(B, Nq, H, D).astype(np.float32), want)


@pytest.mark.gpu
@pytest.mark.parametrize("Nq", [1, 40])
def test_far_keys(hip, Nq):
    """Keys whose offsets pass 2^31 elements (and 4 GiB)."""
    from aria_amd.device import DeviceArray as DA, sync
    L = hip.lib()
    r = rng(31)
    H, Nk, D, far = 2, 70, 64, 1 << 26
    q, k, v = (randn(r, (1, H, n, D)).astype(np.float16) for n in (Nq, Nk, Nk))
    want = run(hip, "f16", q, k, v)
    base = DA((((Nk - 1) * far + 2 * H * D) * 2,), np.uint8)
    kv = np.ascontiguousarray(np.concatenate([k, v], 1)[0].transpose(1, 0, 2))     # [Nk, 2H, D]
    for j in range(Nk):
        L.aria_cuda_memcpy_h2d(base.p + j * far * 2, kv[j].ctypes.data, kv[j].nbytes)
    a = describe(hip, "f16", 1, H, H, Nq, Nk, D)
    dq, do = DA.from_host(q), DA((1, Nq, H * D), np.float16)
    a.q, a.k, a.v, a.out = dq.p, base.p, base.p + H * D * 2, do.p
    a.k_token = a.v_token = far
    a.k_head = a.v_head = D
    ws = DA(max(1, L.aria_hip_cross_attention_ws_bytes(a)), np.uint8)
    hip.check(L.aria_hip_cross_attention_dev(a, ws.p, None))
    sync()
    assert np.array_equal(do.to_host().reshape(1, Nq, H, D).astype(np.float32), want)


@pytest.mark.gpu
def test_long_keys_one_query(hip):
    """A single token over encoder states of 20000 tokens, ragged, and a masked one."""
    lens = [20000, 1, 0, 12345, 8193]
    check(hip, "bf16", 5, 4, 1, 1, 20000, 64, 41, kv_len=lens)
    mask = (rng(2).random((5, 20000)) < 0.3).astype(np.uint8)
    mask[0, :16000] = 0
    check(hip, "f16", 5, 4, 1, 2, 20000, 128, 42, kv_len=lens, mask=mask)


@pytest.mark.gpu
def test_host_form(hip):
    from aria_amd import ops
    r = rng(51)
    q, k, v = (randn(r, s) for s in ((2, 4, 20, 64), (2, 2, 77, 64), (2, 2, 77, 64)))
    f = [x.astype(np.float16).astype(np.float32) for x in (q, k, v)]
    mask = r.random((2, 77)) < 0.6
    got = ops.cross_attention(q, k, v, kv_len=[77, 30], mask=mask)
    want, mag = mx4.cross_attention(*f, [77, 30], mask)
    tol = tolerance(want, mag, *f, "f16", "f32", 1 / 8, 77)
    assert (np.abs(got.reshape(want.shape) - want) <= tol).all()
    assert (ops.cross_attention(q, k[:, :, :0], v[:, :, :0]) == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("Nq,Nk", [(1, 9000), (200, 300)])
def test_two_streams(hip, Nq, Nk):
    """Two calls at once on streams and workspaces of their own give the bits of each alone."""
    from aria_amd.device import DeviceArray as DA
    L = hip.lib()
    r = rng(61)
    H, D = 4, 64
    data = [[randn(r, (1, H, n, D)).astype(np.float16) for n in (Nq, Nk, Nk)] for _ in range(2)]
    want = [run(hip, "f16", *x) for x in data]
    st = [L.aria_hip_stream_create() for _ in data]
    keep, outs = [], []
    try:
        calls = []
        for x in data:
            a = describe(hip, "f16", 1, H, H, Nq, Nk, D)
            d = [DA.from_host(y) for y in x]
            do = DA((1, Nq, H * D), np.float16)
            a.q, a.k, a.v, a.out = d[0].p, d[1].p, d[2].p, do.p
            ws = DA(max(1, L.aria_hip_cross_attention_ws_bytes(a)), np.uint8)
            keep += [d, ws]
            outs.append(do)
            calls.append((a, ws))
        for _ in range(5):
            for i, (a, ws) in enumerate(calls):
                hip.check(L.aria_hip_cross_attention_dev(a, ws.p, st[i]))
        for s in st:
            hip.check(L.aria_hip_stream_sync(s))
    finally:
        for s in st:
            L.aria_hip_stream_destroy(s)
    for o, w in zip(outs, want):
        assert np.array_equal(o.to_host().reshape(w.shape).astype(np.float32), w)
