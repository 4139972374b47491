"""Attention of a batch over shared prefixes and own keys in the 8-bit cache through the C ABI, against the
definition in 64 bits (oracle/states.py). Refusals run on the CPU."""
from __future__ import annotations

import numpy as np
import pytest

from conftest import randn, rng
from oracle import mx4, states
from test_states import Cache, back, cast, dev, ptr
from test_cross_attn import tolerance
from test_mx4_layer import replayed

CODE = {"f16": 1, "bf16": 2}
P = 4096     # never dereferenced


def describe(hip, t, B, H, Nq, D, prefix, own, layout="heads", scale=None):
    a = hip.PrefixAttention(prefix=prefix, own=own, type=CODE[t], B=B, H=H, Nq=Nq, scale=1 / np.sqrt(D) if scale is None else scale,
                            o_batch=Nq * H * D, o_token=H * D, o_head=D)
    if layout == "heads":
        a.q_batch, a.q_head, a.q_token = H * Nq * D, Nq * D, D
    else:
        a.q_batch, a.q_token, a.q_head = Nq * H * D, H * D, D
    return a


# ---- CPU ----

def test_refusals():
    import aria_amd
    L = aria_amd.lib()

    def call(ws=P, prefix={}, own={}, **kw):
        caches = []
        for b, more in ((2, prefix), (4, own)):
            c = aria_amd.KVCache(k=P, v=P, k_scale=P, v_scale=P, batch=4096, head=1024, token=64, s_batch=32, s_head=16, B=b, Hkv=2,
                                 D=64, cap=16)
            for n, v in more.items():
                setattr(c, n, v)
            caches.append(c)
        a = describe(aria_amd, "f16", 4, 8, 3, 64, *caches)
        a.q = a.out = P
        for n, v in kw.items():
            setattr(a, n, v)
        return L.aria_hip_prefix_attention_dev(a, ws, None), L.aria_hip_prefix_attention_ws_bytes(a)
    for kw in (dict(H=3), dict(H=0), dict(B=3), dict(B=-1), dict(Nq=-1), dict(prefix=dict(B=3)), dict(prefix=dict(B=0)),
               dict(own=dict(B=2)), dict(prefix=dict(Hkv=4)), dict(own=dict(Hkv=0)), dict(prefix=dict(D=128)),
               dict(prefix=dict(D=24), own=dict(D=24)), dict(prefix=dict(D=144), own=dict(D=144)), dict(prefix=dict(cap=-1)),
               dict(own=dict(cap=-1)), dict(Nq=1 << 26), dict(B=1 << 18, own=dict(B=1 << 18))):
        assert call(**kw) == (-1, 0), kw
        assert "invalid argument" in aria_amd.last_error()
    for kw in (dict(type=0), dict(type=3), dict(q=None), dict(out=None), dict(q=P + 8), dict(out=P + 2), dict(q_head=4), dict(o_token=-8),
               dict(q_batch=12), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
               dict(prefix_len=P + 1), dict(own_len=P + 2), dict(first=P + 3), dict(prefix=dict(k=None)), dict(own=dict(v_scale=None)),
               dict(own=dict(v=P + 8)), dict(prefix=dict(token=72)), dict(own=dict(head=-16)), dict(ws=P + 8)):
        assert call(**kw)[0] == -1, kw
    assert call(B=0, own=dict(B=0), q=None)[0] == 0 and call(Nq=0, out=None)[0] == 0
    assert L.aria_hip_prefix_attention_dev(None, None, None) == -1 and L.aria_hip_prefix_attention_ws_bytes(None) == 0


# ---- GPU ----

def fill(hip, r, B, h, cap, D, tokens_first=False, spread=1.0):
    """A cache of random rows, scales of their own to each row; its values as (k, v) [B, h, cap, D] in 64 bits"""
    c = Cache(hip, B, h, max(cap, 1), D, tokens_first)
    out = []
    for i in range(2):
        x = randn(r, (B, cap, h, D)) * (spread if i == 0 else 1) * np.exp2(r.integers(-2, 2, (B, cap, h, 1)))
        code, byte = states.rows(x.astype(np.float32))
        if cap:
            c.put(i, code, byte)
        out.append(states.values(code, byte).transpose(0, 2, 1, 3))
    c.c.cap = cap
    return c, out


def poison(c, hidden):
    """Rows of the mask `hidden` [B, cap] become NaN (byte 255)"""
    for i in range(2):
        code, byte = (x.copy() for x in c.get(i))
        code[hidden], byte[hidden] = 0x7F, 255
        c.put(i, code, byte)


def run(hip, t, q, prefix, own, prefix_len=None, own_len=None, first=None, out="same", layout="heads", scale=None, stream=None):
    """q [B, H, Nq, D] in the type; caches; -> [B, Nq, H, D]"""
    from aria_amd.device import DeviceArray as DA, sync
    L = hip.lib()
    B, H, Nq, D = q.shape
    a = describe(hip, t, B, H, Nq, D, prefix.c, own.c, layout, scale)
    dq = DA.from_host(q if layout == "heads" else np.ascontiguousarray(q.transpose(0, 2, 1, 3)))
    guard = 2
    do = DA.from_host(np.full((B * Nq + guard, H * D), 99, np.float32 if out == "f32" else q.dtype))
    a.q, a.out, a.out_f32 = dq.p, do.p, int(out == "f32")
    d = [dev(x) for x in (prefix_len, own_len, first)]
    a.prefix_len, a.own_len, a.first = (ptr(x) for x in d)
    ws = DA(max(1, L.aria_hip_prefix_attention_ws_bytes(a)) + 256, np.uint8)
    ws.upload(np.full(ws.shape, 0xFF, np.uint8))
    hip.check(L.aria_hip_prefix_attention_dev(a, ws.p, stream))
    sync(stream)
    o = do.to_host()
    assert (o[B * Nq:] == 99).all(), "rows behind the last one were written"
    assert (ws.to_host()[-256:] == 0xFF).all(), "written behind the workspace"
    return back(o[:B * Nq].reshape(B, Nq, H, D), "f32" if out == "f32" else t)


def check(hip, t, B, Pn, H, Hkv, Nq, n, m, D, seed, ragged=False, causal=False, out="same", layout="heads", tokens_first=False,
          hide=False):
    r = rng(seed)
    print(f"[gpu] prefix attention {t} B {B}/{Pn} H {H}/{Hkv} Nq {Nq} keys {n} + {m} D {D} ragged {ragged} causal {causal}", flush=True)
    q, qv = cast(randn(r, (B, H, Nq, D)), t)
    cp, pv = fill(hip, r, Pn, Hkv, n, D, tokens_first)
    co, ov = fill(hip, r, B, Hkv, m, D, not tokens_first)
    pl = r.integers(0, n + 1, Pn) if ragged else None
    ol = r.integers(0, m + 1, B) if ragged else None
    if ragged and B > 2:
        ol[1], ol[2] = 0, m
    first = None
    if causal:                               # the last Nq of the own slots, some sequences with more queries than slots
        first = (np.full(B, m) if ol is None else ol) - Nq
    if hide:
        if pl is not None and n:
            poison(cp, np.arange(n)[None] >= pl[:, None])
        if ol is not None and m:
            poison(co, np.arange(m)[None] >= ol[:, None])
    got = run(hip, t, q, cp, co, pl, ol, first, out, layout)
    want, mag = states.attention(qv, pv, ov, pl, ol, first)
    # the cache's values are exact in both types here; tolerance() states the derivation
    k = np.concatenate((pv[0].ravel(), ov[0].ravel()))
    v = np.concatenate((pv[1].ravel(), ov[1].ravel()))
    tol = tolerance(want, mag, qv, k, v, t, out if out == "f32" else t, 1 / np.sqrt(D), n + m)
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) - tol).max()
    return got


SHAPES = [
    # B, prefixes, H, Hkv, Nq, prefix, own, D
    (1, 1, 1, 1, 1, 1, 0, 64), (1, 1, 1, 1, 1, 0, 1, 128), (2, 1, 4, 2, 1, 33, 5, 64), (4, 2, 4, 1, 3, 70, 31, 128), (6, 3, 2, 2, 5, 64, 64, 80),
    (3, 1, 4, 4, 33, 129, 40, 64), (2, 2, 2, 2, 130, 65, 200, 64), (2, 1, 4, 2, 70, 31, 33, 128), (8, 1, 4, 1, 1, 700, 90, 128),
    (2, 1, 2, 1, 1, 3000, 7, 64), (5, 5, 2, 1, 9, 40, 300, 96), (4, 4, 1, 1, 150, 257, 1, 32), (33, 1, 4, 2, 2, 130, 9, 64),
    (2, 1, 8, 8, 140, 100, 140, 128), (16, 4, 16, 16, 40, 90, 20, 64), (2, 1, 2, 2, 3, 0, 0, 64), (3, 3, 2, 1, 1, 1030, 0, 16),
    (32, 1, 16, 16, 17, 257, 0, 64), (9, 1, 16, 8, 30, 70, 70, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("B,Pn,H,Hkv,Nq,n,m,D", [(6, 1, 8, 8, 710, 8716, 250, 64), (11, 1, 8, 4, 388, 9001, 0, 64),
                                                 (6, 2, 8, 4, 134, 16001, 291, 32), (3, 1, 32, 8, 437, 5001, 700, 128)])
def test_splits_in_several_rounds(hip, B, Pn, H, Hkv, Nq, n, m, D):
    """Many rows over long keys: more workgroups than the CUs hold at once, whose results are joined."""
    r = rng(B * Nq + n)
    print(f"[gpu] prefix attention f16 B {B}/{Pn} H {H}/{Hkv} Nq {Nq} keys {n} + {m} D {D}", flush=True)
    q, qv = cast(randn(r, (B, H, Nq, D)), "f16")
    cp, pv = fill(hip, r, Pn, Hkv, n, D)
    co, ov = fill(hip, r, B, Hkv, m, D)
    pl, ol = np.full(Pn, n - 5), r.integers(0, m + 1, B)
    first = ol - Nq // 2
    got = run(hip, "f16", q, cp, co, pl, ol, first, "f32")
    G = H // Hkv
    for b, h in ((0, 0), (B - 1, H - 1)):        # two heads of them all
        p, k = b * Pn // B, h // G
        one = [x[p:p + 1, k:k + 1] for x in pv], [x[b:b + 1, k:k + 1] for x in ov]
        want, mag = states.attention(qv[b:b + 1, h:h + 1], *one, pl[p:p + 1], ol[b:b + 1], first[b:b + 1])
        kk, vv = (np.concatenate((one[0][i].ravel(), one[1][i].ravel())) for i in range(2))
        tol = tolerance(want, mag, qv[b:b + 1, h:h + 1], kk, vv, "f16", "f32", 1 / np.sqrt(D), n + m)
        assert (np.abs(got[b:b + 1, :, h:h + 1] - want) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(hip, t, shape):
    for i, (ragged, causal) in enumerate(((False, False), (True, False), (False, True), (True, True))):
        check(hip, t, *shape, seed=sum(shape) + i, ragged=ragged, causal=causal, out=("same", "f32")[i % 2], layout=("heads", "tokens")[i // 2],
              tokens_first=bool(i % 2), hide=ragged)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 1, 4, 2, 1, 40, 40, 64), (3, 3, 4, 2, 20, 33, 70, 128), (2, 1, 4, 4, 150, 70, 160, 64)])
def test_nan_that_a_row_sees(hip, shape):
    """A row of byte 255 reaches the rows that see it, whole, and no others: keys or values, of the prefix or own, behind a
    causal limit or within it."""
    B, Pn, H, Hkv, Nq, n, m, D = shape
    r = rng(7)
    q, qv = cast(randn(r, (B, H, Nq, D)), "bf16")
    cp, pv = fill(hip, r, Pn, Hkv, n, D)
    co, ov = fill(hip, r, B, Hkv, m, D)
    first = np.full(B, m - Nq)
    clean = run(hip, "bf16", q, cp, co, first=first)
    slot = m - 1 - Nq // 2
    for which in range(2):
        code, byte = (x.copy() for x in co.get(which))
        bad, badb = code.copy(), byte.copy()
        bad[0, slot, 0], badb[0, slot, 0] = 0x7F, 255
        co.put(which, bad, badb)
        got = run(hip, "bf16", q, cp, co, first=first)
        co.put(which, code, byte)
        hit = np.zeros((B, Nq, H), bool)
        hit[0, :, :H // Hkv] = (first[0] + np.arange(Nq) >= slot)[:, None]
        assert hit.any()
        assert np.isnan(got[hit]).all() and np.array_equal(got[~hit], clean[~hit])
    code, byte = (x.copy() for x in cp.get(1))
    bad, badb = code.copy(), byte.copy()
    bad[0, n // 2, Hkv - 1], badb[0, n // 2, Hkv - 1] = 0x7F, 255
    cp.put(1, bad, badb)
    got = run(hip, "bf16", q, cp, co, first=first)
    hit = np.zeros((B, Nq, H), bool)
    hit[:B // Pn, :, H - H // Hkv:] = True
    assert np.isnan(got[hit]).all() and np.array_equal(got[~hit], clean[~hit])


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_large_scores(hip, t):
    """Scores whose steps in fp32 are large: the softmax is that of the largest, ties shared, in every form."""
    for B, Pn, Nq, n, m in ((1, 1, 1, 40, 40), (4, 1, 2, 300, 30), (2, 2, 140, 70, 10)):
        D, H = 64, 2
        q = np.ones((B, H, Nq, D), np.float32)
        q, _ = cast(q, t)
        cp, pv = fill(hip, rng(1), Pn, 1, n, D)
        co, ov = fill(hip, rng(2), B, 1, m, D)
        for c, cap, b, keep in ((cp, n, Pn, pv), (co, m, B, ov)):
            k = np.ones((b, cap, 1, D), np.float32)
            k[:, 5] = 1.0625 if c is cp else 1.0
            k[:, 9] = 1.0625
            code, byte = states.rows(k)
            c.put(0, code, byte)
            keep[0] = states.values(code, byte).transpose(0, 2, 1, 3)
        got = run(hip, t, q, cp, co, scale=2.0 ** 30)
        # 1.0625 is 1 in e4m3 (a tie to the even code): all keys are equal, and all weights
        v = np.concatenate((np.repeat(pv[1], B // Pn, 0), ov[1]), 2)
        want = v.mean(2)[:, None]
        assert np.abs(got - want).max() <= (2 * (2.0 ** -8 if t == "bf16" else 2.0 ** -11) + 2.0 ** -20) * np.abs(v).max()


@pytest.mark.gpu
@pytest.mark.parametrize("Nq,n,m", [(1, 3000, 40), (5, 90, 200), (130, 70, 130)])
def test_captured(hip, Nq, n, m):
    """Shared and not, joined and not, in a graph; lengths are read at each replay."""
    from aria_amd.device import DeviceArray as DA
    L = hip.lib()
    r = rng(Nq)
    B, Pn, H, Hkv, D = 4, 2, 4, 2, 64
    qs = [cast(randn(r, (B, H, Nq, D)), "f16")[0] for _ in range(3)]
    lens = [[[n, n // 2], [m, 0, 3, m], [m - Nq, 0, 1, 5]], [[0, 1], [1, 2, 3, 4], [0, 0, 0, 0]], [[n - 1, 7], [m] * 4, [m - Nq] * 4]]
    cp, co = fill(hip, r, Pn, Hkv, n, D)[0], fill(hip, r, B, Hkv, m, D)[0]
    dq, do, do2 = DA(qs[0].shape, np.float16), *(DA((B, Nq, H * D), np.float16) for _ in range(2))
    dl = [DA((k,), np.int32) for k in (Pn, B, B)]
    a = describe(hip, "f16", B, H, Nq, D, cp.c, co.c)
    a.q, a.out, a.prefix_len, a.own_len, a.first = dq.p, do.p, *(x.p for x in dl)
    ws, ws2 = (DA(max(1, int(L.aria_hip_prefix_attention_ws_bytes(a))), np.uint8) for _ in range(2))
    other = hip.PrefixAttention.from_buffer_copy(a)
    other.out = do2.p

    def feed(i):
        dq.upload(qs[i])
        for d, x in zip(dl, lens[i]):
            d.upload(np.array(x, np.int32))

    def between():
        hip.check(L.aria_hip_prefix_attention_dev(other, ws2.p, None))
        hip.check(L.aria_hip_stream_sync(None))
    replayed(hip, lambda st: hip.check(L.aria_hip_prefix_attention_dev(a, ws.p, st)), feed, [do], between)


@pytest.mark.gpu
def test_steps_of_a_batch(hip):
    """The operators as a program chains them: a common prompt written once, then each sequence's tokens, one and several at a
    time, rotated, cached and attended; each step against the definition on what was cached."""
    from aria_amd.device import DeviceArray as DA, sync
    L = hip.lib()
    r = rng(11)
    B, H, Hkv, D, rot, n, cap, t = 5, 8, 2, 64, 32, 75, 24, "bf16"
    npos = n + cap
    table = [DA((npos, rot // 2)) for _ in range(2)]
    hip.check(L.aria_hip_rotary_table_dev(table[0].p, table[1].p, hip.RotaryScaling(rot=rot, kind=1, base=10000.0, factor=2.0, gain=1.0),
                                          0, npos, None))
    cos, sin = (x.to_host() for x in table) if sync() is None else None
    want = states.table(rot, 0, npos, kind=1, factor=2.0)
    assert max(np.abs(cos - want[0]).max(), np.abs(sin - want[1]).max()) <= 2.0 ** -21
    cp, co = Cache(hip, 1, Hkv, n, D), Cache(hip, B, Hkv, cap, D)
    k, v = (cast(randn(r, (1, n, Hkv, D)), t) for _ in range(2))
    dk, dv = dev(k[0], k[0].dtype), dev(v[0], v[0].dtype)
    w = hip.KVWrite(cache=cp.c, k=dk.p, v=dv.p, cos=table[0].p, sin=table[1].p, type=2, N=n, rot=rot, npos=npos, k_token=Hkv * D, k_head=D,
                    v_token=Hkv * D, v_head=D)
    hip.check(L.aria_hip_kv_write_dev(w, None))
    held = np.array([0, 0, 0, 0, 0])
    keys = [np.zeros((B, cap, Hkv, D)), np.zeros((B, cap, Hkv, D))]
    for N in (7, 1, 1, 4):
        count = np.minimum(N, [N, max(1, N - 3), N, 0, 1])
        row = (H + 2 * Hkv) * D
        x, xv = cast(randn(r, (B, N, H + 2 * Hkv, D)), t)
        dx, dq, do = dev(x, x.dtype), DA((B, H, N, D), x.dtype), DA((B, N, H, D), x.dtype)
        dq.upload(np.zeros(dq.shape, x.dtype))
        df, dn, dp = dev(held), dev(count), dev(n + held[:, None] + np.arange(N))
        dl = dev(held + count)
        w = hip.KVWrite(cache=co.c, q=dx.p, k=dx.p + 2 * H * D, v=dx.p + 2 * (H + Hkv) * D, q_out=dq.p, cos=table[0].p, sin=table[1].p,
                        pos=dp.p, first=df.p, count=dn.p, pos_stride=N, type=2, N=N, Hq=H, rot=rot, npos=npos, qo_batch=H * N * D, qo_head=N * D, qo_token=D)
        for s in "qkv":
            for axis, st in (("batch", N * row), ("token", row), ("head", D)):
                setattr(w, f"{s}_{axis}", st)
        a = describe(hip, t, B, H, N, D, cp.c, co.c)
        a.q, a.out, a.own_len, a.first = dq.p, do.p, dl.p, df.p
        ws = DA(max(1, int(L.aria_hip_prefix_attention_ws_bytes(a))), np.uint8)
        hip.check(L.aria_hip_kv_write_dev(w, None))
        hip.check(L.aria_hip_prefix_attention_dev(a, ws.p, None))
        sync()
        # the cache holds each sequence's tokens, rotated behind the prompt's
        at = n + held[:, None] + np.arange(N)
        rk, _ = states.rotate(xv[:, :, H:H + Hkv], cos[at][:, :, None], sin[at][:, :, None], False)
        for i, y in ((0, rk.astype(np.float32)), (1, xv[:, :, H + Hkv:])):
            val = states.values(*states.rows(y))
            for b in range(B):
                keys[i][b, held[b]:held[b] + count[b]] = val[b, :count[b]]
            got = states.values(*co.get(i))
            for b in range(B):
                assert np.array_equal(got[b, :held[b] + count[b]], keys[i][b, :held[b] + count[b]])
        qv = mx4.bf16_value(dq.to_host())
        pk = [states.values(*cp.get(i)).transpose(0, 2, 1, 3) for i in range(2)]
        ok = [x.transpose(0, 2, 1, 3) for x in keys]
        want, mag = states.attention(qv, pk, ok, None, held + count, held)
        got = mx4.bf16_value(do.to_host())
        kk, vv = (np.concatenate((pk[i].ravel(), ok[i].ravel())) for i in range(2))
        tol = tolerance(want, mag, qv, kk, vv, t, t, 1 / np.sqrt(D), n + cap)
        told = np.arange(N)[None] < count[:, None]
        assert (np.abs(got - want) <= tol)[told].all()
        held = held + count


@pytest.mark.gpu
@pytest.mark.parametrize("Nq", [1, 40])
def test_offsets_past_32_bits(hip, Nq):
    """Sequences, heads and slots that lie further apart than 2^32 bytes: written, read and attended."""
    from aria_amd.device import DeviceArray as DA, sync
    L = hip.lib()
    r = rng(Nq)
    B, H, Hkv, D, n = 2, 2, 2, 64, 70
    token, head, batch = 1 << 23, 1 << 30, (1 << 32) + (1 << 31) + 4096
    size = batch + head + (n - 1) * token + D
    code, byte = [DA((size,), np.uint8) for _ in range(2)], [DA((B * Hkv * n,), np.uint8) for _ in range(2)]
    c = hip.KVCache(k=code[0].p, v=code[1].p, k_scale=byte[0].p, v_scale=byte[1].p, B=B, Hkv=Hkv, D=D, cap=n, batch=batch, head=head,
                    token=token, s_batch=Hkv * n, s_head=n)
    x = [cast(randn(r, (B, n, Hkv, D)), "bf16") for _ in range(2)]
    dx = [dev(a[0], a[0].dtype) for a in x]
    w = hip.KVWrite(cache=c, k=dx[0].p, v=dx[1].p, type=2, N=n)
    back_ = [DA((B, n, Hkv, D)) for _ in range(2)]
    a = hip.KVRead(cache=c, k=back_[0].p, v=back_[1].p, type=0, N=n)
    for s in "kv":
        for d in (w, a):
            for axis, st in (("batch", n * Hkv * D), ("token", Hkv * D), ("head", D)):
                setattr(d, f"{s}_{axis}", st)
    hip.check(L.aria_hip_kv_write_dev(w, None))
    hip.check(L.aria_hip_kv_read_dev(a, None))
    sync()
    held = [states.values(*states.rows(v)) for _, v in x]
    assert all(np.array_equal(b.to_host(), h) for b, h in zip(back_, held))
    q, qv = cast(randn(r, (B, H, Nq, D)), "bf16")
    none = hip.KVCache(B=B, Hkv=Hkv, D=D)

    class As:
        def __init__(self, c):
            self.c = c
    pv = [h.transpose(0, 2, 1, 3) for h in held]
    no = [np.zeros((B, Hkv, 0, D))] * 2
    for prefix, own, p, o in ((c, none, pv, no), (none, c, no, pv)):
        got = run(hip, "bf16", q, As(prefix), As(own))
        want, mag = states.attention(qv, p, o)
        assert (np.abs(got - want) <= tolerance(want, mag, qv, pv[0], pv[1], "bf16", "bf16", 1 / np.sqrt(D), n)).all()
    for d in code:
        d.free()


@pytest.mark.gpu
def test_two_streams_and_repeats(hip):
    """Calls in flight on two streams with a workspace each, and the same call again: the same bits."""
    from aria_amd.device import DeviceArray as DA
    L = hip.lib()
    r = rng(21)
    jobs = []
    for B, Pn, H, Hkv, Nq, n, m, D in ((16, 1, 8, 2, 2, 900, 60, 64), (6, 2, 4, 4, 50, 300, 90, 128)):
        cp, co = fill(hip, r, Pn, Hkv, n, D)[0], fill(hip, r, B, Hkv, m, D)[0]
        q = cast(randn(r, (B, H, Nq, D)), "f16")[0]
        a = describe(hip, "f16", B, H, Nq, D, cp.c, co.c)
        dq, do = DA.from_host(q), DA((B, Nq, H, D), np.float16)
        a.q, a.out = dq.p, do.p
        jobs.append((a, do, DA(max(1, int(L.aria_hip_prefix_attention_ws_bytes(a))), np.uint8), (cp, co, dq)))
    want = []
    for a, do, ws, _ in jobs:
        hip.check(L.aria_hip_prefix_attention_dev(a, ws.p, None))
        hip.check(L.aria_hip_stream_sync(None))
        want.append(do.to_host())
        do.upload(np.zeros(do.shape, do.dtype))
    st = [L.aria_hip_stream_create() for _ in jobs]
    for _ in range(5):
        for s, (a, _, ws, _) in zip(st, jobs):
            hip.check(L.aria_hip_prefix_attention_dev(a, ws.p, s))
    for s, (_, do, _, _), w in zip(st, jobs, want):
        hip.check(L.aria_hip_stream_sync(s))
        assert do.to_host().tobytes() == w.tobytes()
        L.aria_hip_stream_destroy(s)
