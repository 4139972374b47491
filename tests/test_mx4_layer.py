"""GPU: a text-conditioned layer with MXFP4 weights as a program chains it: norm -> q projection -> head
preparation; context -> k/v projection -> head preparation; cross attention over prompts of different
lengths; output projection, gated residual; norm -> gated up-projection -> down projection -> residual.
Every new operator's output is checked against its definition in 64 bits on the inputs that it had, and
the chain captured into a HIP graph gives the eager chain's bits on every replay."""
from __future__ import annotations

import ctypes as C
import os

import numpy as np
import pytest

from conftest import ROOT, randn, rng
from oracle import mx4
from test_cross_attn import tolerance
from test_mx4 import linear_tol

pytestmark = pytest.mark.gpu

B, S, H, DIM, CTX, NK, INNER = 2, 70, 4, 256, 192, 50, 320
LENS = [50, 13]


class Layer:
    def __init__(self, hip, seed):
        from aria_amd.device import DeviceArray as DA
        r = rng(seed)
        self.hip, self.L = hip, hip.lib()
        self.w = {n: mx4.quant(randn(r, shape, 1 / np.sqrt(shape[1]))) for n, shape in
                  dict(q=(DIM, DIM), kv=(2 * DIM, CTX), o=(DIM, DIM), up=(2 * INNER, DIM), down=(DIM, INNER)).items()}
        self.b = randn(r, 2 * INNER, 0.1)
        self.dw = {n: (DA.from_host(q), DA.from_host(s)) for n, (q, s) in self.w.items()}
        self.db = DA.from_host(self.b)
        self.gain = DA.from_host(np.ones(DIM, np.float32))
        self.gate = DA.from_host(randn(r, (B, DIM)))
        self.lens = DA.from_host(np.array(LENS, np.int32))
        M, MK = B * S, B * NK
        f32, f16 = np.float32, np.float16
        self.d = {n: DA(shape, t) for n, (shape, t) in dict(
            x=((M, DIM), f32), ctx=((MK, CTX), f32), n1=((M, DIM), f32), qp=((M, DIM), f32), kvp=((MK, 2 * DIM), f32),
            q=((B, H, S, 64), f16), k=((B, H, NK, 64), f16), v=((B, H, NK, 64), f16), a=((B, S, DIM), f16),
            o=((M, DIM), f32), r=((M, DIM), f32), n2=((M, DIM), f32), h=((M, INNER), f16), f=((M, DIM), f32),
            y=((M, DIM), f32)).items()}
        # one workspace for all: the chain's calls run one after another on their stream
        self.ws = DA(int(max(self.L.aria_hip_mx4_ws_bytes(M, k) for k in (DIM, CTX, INNER))), np.uint8)
        a = self.att = hip.CrossAttention(type=1, B=B, H=H, Hkv=H, Nq=S, Nk=NK, D=64, scale=0.125, kv_len=self.lens.p,
                                          q=self.d["q"].p, k=self.d["k"].p, v=self.d["v"].p, out=self.d["a"].p,
                                          q_batch=H * S * 64, q_head=S * 64, q_token=64, k_batch=H * NK * 64, k_head=NK * 64,
                                          k_token=64, v_batch=H * NK * 64, v_head=NK * 64, v_token=64, o_batch=S * DIM,
                                          o_head=64, o_token=DIM)
        self.aws = DA(max(1, int(self.L.aria_hip_cross_attention_ws_bytes(a))), np.uint8)

    def run(self, st):
        L, d, M, MK = self.L, self.d, B * S, B * NK
        ck = self.hip.check

        def lin(y, yt, x, xt, name, m, k, n, bias=None, fn="aria_hip_linear_mx4_dev"):
            q, s = self.dw[name]
            ck(getattr(L, fn)(d[y].p, yt, d[x].p, xt, k, q.p, s.p, bias, m, k, n, self.ws.p, st), name)

        def heads(src, secs, s, kinds):
            ck(L.aria_hip_qkv_prep_dev(d[src].p, len(secs) * DIM, B, s, H, len(secs), (C.c_int * 3)(*kinds),
                                       (C.c_void_p * 3)(*[d[n].p for n in secs]), (C.c_void_p * 3)(None, None, None),
                                       None, None, 0, 1e-6, st), src)

        ck(L.aria_hip_rmsnorm_dev(d["n1"].p, d["x"].p, self.gain.p, M, DIM, 1e-5, st))
        lin("qp", 0, "n1", 0, "q", M, DIM, DIM)
        heads("qp", ["q"], S, [0])
        lin("kvp", 0, "ctx", 0, "kv", MK, CTX, 2 * DIM)
        heads("kvp", ["k", "v"], NK, [1, 2])
        ck(L.aria_hip_cross_attention_dev(self.att, self.aws.p, st))
        lin("o", 0, "a", 1, "o", M, DIM, DIM)
        ck(L.aria_hip_gate_residual_dev(d["r"].p, d["x"].p, d["o"].p, self.gate.p, None, M, DIM, S, st))
        ck(L.aria_hip_rmsnorm_dev(d["n2"].p, d["r"].p, self.gain.p, M, DIM, 1e-5, st))
        lin("h", 1, "n2", 0, "up", M, DIM, INNER, self.db.p, "aria_hip_glu_mx4_dev")
        lin("f", 0, "h", 1, "down", M, INNER, DIM)
        ck(L.aria_hip_add_dev(d["y"].p, d["r"].p, d["f"].p, M * DIM, st))

    def feed(self, x, ctx):
        self.d["x"].upload(x)
        self.d["ctx"].upload(ctx)


def test_layer(hip):
    layer = Layer(hip, 5)
    r = rng(6)
    layer.feed(randn(r, (B * S, DIM)), randn(r, (B * NK, CTX)))
    layer.run(None)
    hip.check(hip.lib().aria_hip_stream_sync(None))
    v = {n: a.to_host().astype(np.float32) for n, a in layer.d.items()}
    for y, x, name, k in (("qp", "n1", "q", DIM), ("kvp", "ctx", "kv", CTX), ("o", "a", "o", DIM), ("f", "h", "down", INNER)):
        want, terms = mx4.linear(v[x].reshape(-1, k), *layer.w[name])
        assert (np.abs(v[y] - want) <= linear_tol(want, terms, k, "f32")).all(), name
    want, mag = mx4.cross_attention(v["q"], v["k"], v["v"], LENS)
    tol = tolerance(want, mag, v["q"], v["k"], v["v"], "f16", "f16", 0.125, NK)
    assert (np.abs(v["a"].reshape(B, S, H, 64) - want) <= tol).all()
    lin, terms = mx4.linear(v["n2"], *layer.w["up"], layer.b)
    val, g = lin[:, :INNER], lin[:, INNER:]
    want = val * g / (1 + np.exp(-g))
    d = linear_tol(0 * lin, terms, DIM, "f32")
    tol = np.abs(g) * d[:, :INNER] + 1.1 * np.abs(val) * d[:, INNER:] + (8 + np.abs(g)) * 2.0 ** -23 * np.abs(want)
    assert (np.abs(v["h"] - want) <= tol + 2.0 ** -11 * np.abs(want) * 1.001 + 2.0 ** -25).all()
    assert np.array_equal(v["y"], v["r"] + v["f"])


def probe():
    P = C.CDLL(os.path.join(ROOT, "aria_amd", "libaria_probe.so"))
    for name, args in (("aria_probe_capture_begin", [C.c_void_p]), ("aria_probe_capture_end", [C.c_void_p, C.POINTER(C.c_void_p)]),
                       ("aria_probe_graph_launch", [C.c_void_p, C.c_void_p]), ("aria_probe_graph_free", [C.c_void_p])):
        getattr(P, name).restype, getattr(P, name).argtypes = C.c_int, args
    return P


def replayed(hip, run, feed, outputs, eager_between):
    """``run`` captured once; each replay on new inputs against the eager run's outputs, with eager work between."""
    L, P = hip.lib(), probe()
    st = L.aria_hip_stream_create()
    ex = C.c_void_p()
    try:
        want = []
        for i in range(3):
            feed(i)
            run(None)
            hip.check(L.aria_hip_stream_sync(None))
            want.append([o.to_host() for o in outputs])
        assert P.aria_probe_capture_begin(st) == 0
        run(st)
        assert P.aria_probe_capture_end(st, C.byref(ex)) == 0 and ex.value
        for i in (0, 1, 2, 1, 0):
            feed(i)
            eager_between()
            for o in outputs:
                o.upload(np.zeros(o.shape, o.dtype))
            assert P.aria_probe_graph_launch(ex, st) == 0
            hip.check(L.aria_hip_stream_sync(st))
            for o, w in zip(outputs, want[i]):
                assert o.to_host().tobytes() == w.tobytes(), f"replay of input {i}"
    finally:
        if ex.value:
            P.aria_probe_graph_free(ex)
        L.aria_hip_stream_destroy(st)


def test_layer_captured(hip):
    layer, other = Layer(hip, 7), Layer(hip, 8)
    r = rng(9)
    data = [(randn(r, (B * S, DIM)), randn(r, (B * NK, CTX))) for _ in range(4)]
    other.feed(*data[3])

    def between():
        other.run(None)
        hip.check(hip.lib().aria_hip_stream_sync(None))
    replayed(hip, layer.run, lambda i: layer.feed(*data[i]), [layer.d["y"], layer.d["h"], layer.d["a"]], between)


@pytest.mark.parametrize("M", [2, 500])
def test_linear_captured(hip, M):
    """One launch (few rows) and two, alone in a graph."""
    from aria_amd.device import DeviceArray as DA
    L = hip.lib()
    r = rng(M)
    K, N = 256, 300
    q, s = mx4.quant(randn(r, (N, K)))
    xs = [randn(r, (M, K)) for _ in range(3)]
    dq, ds, dx, dy, dz = DA.from_host(q), DA.from_host(s), DA((M, K)), DA((M, N)), DA((M, N))
    ws, ws2 = (DA(int(L.aria_hip_mx4_ws_bytes(M, K)), np.uint8) for _ in range(2))

    def call(y, w, st):
        hip.check(L.aria_hip_linear_mx4_dev(y.p, 0, dx.p, 0, K, dq.p, ds.p, None, M, K, N, w.p, st))
    replayed(hip, lambda st: call(dy, ws, st), lambda i: dx.upload(xs[i]), [dy], lambda: call(dz, ws2, None))


@pytest.mark.parametrize("Nq,Nk", [(1, 3000), (90, 200)])
def test_cross_attention_captured(hip, Nq, Nk):
    """Split keys (two launches through a workspace) and not; lengths read at each replay."""
    from aria_amd.device import DeviceArray as DA
    L = hip.lib()
    r = rng(Nq)
    Bc, Hc, D = 2, 4, 64
    data = [[randn(r, (Bc, Hc, n, D)).astype(np.float16) for n in (Nq, Nk, Nk)] for _ in range(3)]
    lens = [[Nk, 17], [0, Nk // 2], [65, Nk]]
    d = [DA(x.shape, np.float16) for x in data[0]]
    dl, do = DA((Bc,), np.int32), DA((Bc, Nq, Hc * D), np.float16)
    a = hip.CrossAttention(type=1, B=Bc, H=Hc, Hkv=Hc, Nq=Nq, Nk=Nk, D=D, scale=0.125, kv_len=dl.p, q=d[0].p, k=d[1].p, v=d[2].p,
                           out=do.p, q_batch=Hc * Nq * D, q_head=Nq * D, q_token=D, k_batch=Hc * Nk * D, k_head=Nk * D, k_token=D,
                           v_batch=Hc * Nk * D, v_head=Nk * D, v_token=D, o_batch=Nq * Hc * D, o_head=D, o_token=Hc * D)
    ws, ws2 = (DA(max(1, int(L.aria_hip_cross_attention_ws_bytes(a))), np.uint8) for _ in range(2))

    def feed(i):
        for t, x in zip(d, data[i]):
            t.upload(x)
        dl.upload(np.array(lens[i], np.int32))
    other = hip.CrossAttention.from_buffer_copy(a)
    do2 = DA(do.shape, np.float16)
    other.out = do2.p

    def between():
        hip.check(L.aria_hip_cross_attention_dev(other, ws2.p, None))
        hip.check(L.aria_hip_stream_sync(None))
    replayed(hip, lambda st: hip.check(L.aria_hip_cross_attention_dev(a, ws.p, st)), feed, [do], between)
