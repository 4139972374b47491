"""MXFP4 quantisation, product and gated feed-forward through the C ABI, against their definitions in
64 bits (oracle/mx4.py). Refusals and the oracle itself run on the CPU."""
from __future__ import annotations

import numpy as np
import pytest

from conftest import randn, rng
from oracle import mx4

TYPES = ("f32", "f16", "bf16")
CODE = {"f32": 0, "f16": 1, "bf16": 2}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}   # a rounding's largest relative error
SUB = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}      # and its largest absolute one near zero


def cast(x, t):
    """(the array as the device takes it, its values in fp32)"""
    if t == "f32":
        return np.ascontiguousarray(x, np.float32), np.asarray(x, np.float32)
    if t == "f16":
        h = np.asarray(x).astype(np.float16)
        return h, h.astype(np.float32)
    u = mx4.bf16_bits(x)
    return u, mx4.bf16_value(u)


def values(a, t):
    return mx4.bf16_value(a) if t == "bf16" else a.astype(np.float32)


def np_type(t):
    return {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}[t]


# ---- CPU ----

def test_oracle_quantiser_is_nearest():
    """Codes against a search over all sixteen, the lower of two equally near ones where its code is even."""
    r = rng(1)
    x = randn(r, (40, 64)) * np.exp(2 * randn(r, (40, 64)))
    q, s = mx4.quant(x)
    v = mx4.dequant(q, s, 64)
    scale = np.ldexp(1.0, np.repeat(s.astype(int), 32, 1) - 127)
    err = np.abs(np.minimum(np.abs(x) / scale, 6.0)[..., None] - mx4.MAG)
    best = np.abs(np.minimum(np.abs(x.astype(np.float64)) / scale, 6.0) - np.abs(v) / scale)
    assert np.allclose(best, err.min(-1), atol=1e-6)
    ties = np.array([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0] + [0.0] * 24])
    assert (mx4.dequant(*mx4.quant(ties), 32)[0, :8] == [0, 1, 1, 2, 2, 4, 4, 4]).all()


def test_refusals():
    """Each is refused before any device work, by its error code and text."""
    import aria_amd
    L = aria_amd.lib()
    p = 4096   # never dereferenced: the call is refused first

    def bad(rc, what):
        assert rc == -1, rc
        assert what in aria_amd.last_error(), aria_amd.last_error()
    bad(L.aria_hip_mx4_quant_dev(p, p, p, 3, 1, 32, 32, None), "xtype")
    bad(L.aria_hip_mx4_quant_dev(p, p, p, 0, 1, 0, 32, None), "K > 0")
    bad(L.aria_hip_mx4_quant_dev(p, p, p, 0, -1, 32, 32, None), "rows")
    bad(L.aria_hip_mx4_quant_dev(p, p, p, 0, 2, 32, 31, None), "ldx")
    bad(L.aria_hip_mx4_quant_dev(p + 8, p, p, 0, 1, 32, 32, None), "dq")
    bad(L.aria_hip_mx4_quant_dev(p, p, p + 2, 0, 1, 32, 32, None), "dx")
    bad(L.aria_hip_mx4_quant_dev(p, p, p + 1, 1, 1, 32, 32, None), "dx")
    bad(L.aria_hip_mx4_quant_dev(p, None, p, 0, 1, 32, 32, None), "dscale")
    bad(L.aria_hip_mx4_dequant_dev(p, 5, p, p, 1, 32, None), "ytype")
    bad(L.aria_hip_mx4_dequant_dev(p + 1, 1, p, p, 1, 32, None), "dy")
    bad(L.aria_hip_gemm_mx4_dev(p, 0, p, None, p, p, None, 1, 32, 1, None), "dxs")
    bad(L.aria_hip_gemm_mx4_dev(p, 0, p + 4, p, p, p, None, 1, 32, 1, None), "dxq")
    bad(L.aria_hip_gemm_mx4_dev(p, 0, p, p, p, p, p + 2, 1, 32, 1, None), "db")
    bad(L.aria_hip_linear_mx4_dev(p, 0, p, 0, 32, p, p, None, 1, 32, 1, p + 16, None), "dws")
    bad(L.aria_hip_linear_mx4_dev(p, 0, p, 0, 32, p, p, None, 1, 32, 1, None, None), "dws")
    bad(L.aria_hip_linear_mx4_dev(p, 0, p, 7, 32, p, p, None, 1, 32, 1, p, None), "xtype")
    bad(L.aria_hip_linear_mx4_dev(p, 0, p, 0, 16, p, p, None, 1, 32, 1, p, None), "ldx")
    bad(L.aria_hip_glu_mx4_dev(p, 0, p, 0, 32, p, p, None, 1, 32, -1, p, None), "N >= 0")
    bad(L.aria_hip_mx4_quant(None, p, p, 1, 32), "q")
    bad(L.aria_hip_linear_mx4(p, p, p, None, None, 1, 32, 1), "scale")
    assert L.aria_hip_mx4_ws_bytes(0, 32) == 0 and L.aria_hip_mx4_ws_bytes(3, -1) == 0
    assert L.aria_hip_mx4_ws_bytes(3, 33) >= 3 * (2 * 16 + 2)
    # nothing to do is no error, and needs no pointer
    assert L.aria_hip_linear_mx4_dev(None, 0, None, 0, 32, None, None, None, 0, 32, 5, None, None) == 0
    from aria_amd import ops
    with pytest.raises(ValueError):
        ops.linear_mx4(np.zeros((2, 40), np.float32), np.zeros((3, 16), np.uint8), np.zeros((3, 1), np.uint8))
    with pytest.raises(ValueError):
        ops.glu_mx4(np.zeros((2, 32), np.float32), np.zeros((3, 16), np.uint8), np.zeros((3, 1), np.uint8))


# ---- GPU ----

def edge_rows(K):
    """Rows at the format's corners: ties, saturation, signed zeros, subnormals, huge values, Inf, NaN."""
    r = rng(7)
    x = randn(r, (14, K))
    x[0] = 0.0
    x[1] = -0.0
    x[2] = 0.25 * np.arange(K) % 8 - 4
    x[3] = 7.9
    x[4] = (1e-42 * np.arange(K)).astype(np.float32)
    x[5] *= 1e-38
    x[6] *= 1e37
    x[7] = np.where(np.arange(K) % 2, 3.4028234e38, -1e-38)
    x[8, 0] = np.inf
    x[9, K - 1] = np.nan
    x[10, K // 2] = -np.inf
    x[11] = np.ldexp(1.0, -127 + np.arange(K) % 4)
    x[12] = np.ldexp(7.0, -130 - np.arange(K) % 8)
    x[13] = 5.0 * np.ldexp(1.0, np.arange(K) // 32 % 200 - 100)
    return x.astype(np.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [1, 7, 32, 33, 64, 100, 1024])
@pytest.mark.parametrize("t", TYPES)
def test_quant_bits(hip, K, t):
    """Codes and scale bytes, and the values read back, are the definition's to the bit."""
    from aria_amd.device import DeviceArray as DA, sync
    print(f"[gpu] mx4 quant {t} K {K}", flush=True)
    with np.errstate(over="ignore"):
        x, xv = cast(np.concatenate([edge_rows(K), randn(rng(K), (70, K))]), t)
    rows, nb = x.shape[0], (K + 31) // 32
    want_q, want_s = mx4.quant(xv)
    for pad in (0, 8, 5):
        w = np.zeros((rows, K + pad), x.dtype)
        w[:, :K] = x
        w[:, K:] = cast(np.full((rows, pad), 3e4), t)[0]
        dx, dq, ds = DA.from_host(w), DA((rows + 1, 16 * nb), np.uint8), DA((rows + 1, nb), np.uint8)
        dq.upload(np.full((rows + 1, 16 * nb), 0xAB, np.uint8)); ds.upload(np.full((rows + 1, nb), 0xCD, np.uint8))
        hip.check(hip.lib().aria_hip_mx4_quant_dev(dq.p, ds.p, dx.p, CODE[t], rows, K, K + pad, None))
        sync()
        q, s = dq.to_host(), ds.to_host()
        assert np.array_equal(s[:rows], want_s), np.argwhere(s[:rows] != want_s)[:5]
        assert np.array_equal(q[:rows], want_q), np.argwhere(q[:rows] != want_q)[:5]
        assert (q[rows] == 0xAB).all() and (s[rows] == 0xCD).all()
    want = mx4.dequant(want_q, want_s, K)
    for yt in TYPES:
        dy = DA((rows, K), np_type(yt))
        hip.check(hip.lib().aria_hip_mx4_dequant_dev(dy.p, CODE[yt], dq.p, ds.p, rows, K, None))
        sync()
        got = values(dy.to_host(), yt)
        with np.errstate(over="ignore", invalid="ignore"):
            ref = cast(want.astype(np.float32), yt)[1] if yt != "bf16" else want.astype(np.float32)
        assert np.array_equal(np.isnan(got), np.isnan(ref))
        ok = ~np.isnan(ref)
        assert np.array_equal(got[ok], ref[ok]), yt


def run_linear(hip, fn, x, xt, ldx, q, s, b, M, K, N, yt):
    from aria_amd.device import DeviceArray as DA, sync
    L = hip.lib()
    dx, dq, ds = DA.from_host(x), DA.from_host(q), DA.from_host(s)
    db = DA.from_host(b.astype(np.float32)) if b is not None else None
    ws = DA(max(1, L.aria_hip_mx4_ws_bytes(M, K)), np.uint8)
    guard = 3
    dy = DA((M + guard, N), np_type(yt))
    dy.upload(np.full((M + guard, N), 7, np_type(yt)))
    hip.check(getattr(L, fn)(dy.p, CODE[yt], dx.p, CODE[xt], ldx, dq.p, ds.p, db.p if db else None, M, K, N, ws.p, None))
    sync()
    y = dy.to_host()
    assert (y[M:] == np.full((), 7, np_type(yt))).all(), "rows behind the last one were written"
    return values(y[:M], yt)


def linear_tol(y, terms, K, yt):
    """Every product and the 32 sums of a block are exact; an fp32 sum of nb block sums is off by at
    most one step (2^-23) of the partial sum, itself at most sum |terms|, per addition, whatever the
    order; then the output's rounding, and its smallest step near zero."""
    nb = (K + 31) // 32 + 8
    return nb * 2.0 ** -23 * terms + HALF_STEP[yt] * np.abs(y) * 1.001 + SUB[yt]


SHAPES = [(1, 32, 1), (1, 1024, 1024), (2, 1024, 6144), (3, 40, 33), (7, 4096, 130), (16, 96, 64), (17, 64, 48), (31, 2080, 31),
          (33, 1, 5), (40, 33, 700), (65, 256, 257), (100, 4096, 1024), (129, 160, 384), (200, 1000, 200), (344, 1024, 1024),
          (1000, 512, 72)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", SHAPES)
@pytest.mark.parametrize("xt,yt,bias", [("f32", "f32", True), ("f16", "f16", False), ("bf16", "bf16", True),
                                        ("f16", "f32", True)])
def test_linear(hip, M, K, N, xt, yt, bias):
    print(f"[gpu] linear_mx4 {M} {K} {N} {xt} {yt}", flush=True)
    r = rng(M * 7 + K + N)
    x, xv = cast(randn(r, (M, K)) * np.exp(0.5 * randn(r, (1, K))), xt)
    q, s = mx4.quant(randn(r, (N, K), 0.02))
    b = randn(r, N, 0.5) if bias else None
    y, terms = mx4.linear(xv, q, s, b)
    got = run_linear(hip, "aria_hip_linear_mx4_dev", x, xt, K, q, s, b, M, K, N, yt)
    assert (np.abs(got - y) <= linear_tol(y, terms, K, yt)).all(), np.abs(got - y).max()


LARGE = [(900, 480, 1501), (900, 1000, 1500), (1500, 1024, 2050), (2592, 1056, 3500), (2700, 1111, 4090),
         (1000, 2500, 2100), (4090, 2111, 4095)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", LARGE)
@pytest.mark.parametrize("xt,yt,bias", [("f32", "f32", True), ("bf16", "f16", False)])
def test_linear_large(hip, M, K, N, xt, yt, bias):
    """Tiles of 64, 128 and 256 rows, whole and cut at every edge, K in whole chunks and not."""
    test_linear(hip, M, K, N, xt, yt, bias)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 5, 60, 300])
@pytest.mark.parametrize("pad", [8, 3])
def test_linear_row_stride(hip, M, pad):
    """Activations that are a section of wider rows, aligned and not; what lies between does not count."""
    r = rng(M + pad)
    K, N = 200, 77
    w = np.full((M, K + pad), np.nan, np.float32)
    w[:, :K] = randn(r, (M, K))
    q, s = mx4.quant(randn(r, (N, K)))
    y, terms = mx4.linear(w[:, :K], q, s)
    got = run_linear(hip, "aria_hip_linear_mx4_dev", w, "f32", K + pad, q, s, None, M, K, N, "f32")
    assert (np.abs(got - y) <= linear_tol(y, terms, K, "f32")).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [(1, 32, 1), (2, 1024, 4096), (5, 100, 37), (16, 512, 200), (40, 1024, 96), (172, 1024, 520),
                                   (300, 320, 130)])
@pytest.mark.parametrize("xt,yt,bias", [("f32", "f32", True), ("f16", "f16", False), ("bf16", "bf16", True)])
def test_glu(hip, M, K, N, xt, yt, bias):
    print(f"[gpu] glu_mx4 {M} {K} {N} {xt} {yt}", flush=True)
    r = rng(M * 3 + K + N)
    x, xv = cast(randn(r, (M, K)), xt)
    q, s = mx4.quant(randn(r, (2 * N, K), 2 / np.sqrt(K)))
    b = randn(r, 2 * N, 0.5) if bias else None
    lin, terms = mx4.linear(xv, q, s, b)
    v, g = lin[:, :N], lin[:, N:]
    sg = 1 / (1 + np.exp(-g))
    y = v * g * sg
    d = ((K + 31) // 32 + 8) * 2.0 ** -23 * terms
    # v and g are off by d; |d silu / dg| <= 1.1; exp, rcp and three products: |g| 2^-23 (the exponent's
    # rounding) and a step each
    tol = np.abs(g * sg) * d[:, :N] + 1.1 * np.abs(v) * d[:, N:] + (8 + np.abs(g)) * 2.0 ** -23 * np.abs(y)
    tol += HALF_STEP[yt] * np.abs(y) * 1.001 + SUB[yt]
    got = run_linear(hip, "aria_hip_glu_mx4_dev", x, xt, K, q, s, b, M, K, N, yt)
    assert (np.abs(got - y) <= tol).all(), np.abs(got - y).max()


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [(260, 1000, 2050), (520, 700, 1030), (1300, 416, 2050), (2700, 416, 4090), (1000, 2500, 2100),
                                   (4090, 2111, 2047)])
@pytest.mark.parametrize("xt,yt,bias", [("f32", "f32", True), ("f16", "bf16", False)])
def test_glu_large(hip, M, K, N, xt, yt, bias):
    test_glu(hip, M, K, N, xt, yt, bias)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [(260, 1700, 2570), (1100, 300, 1550), (1500, 300, 3085), (1900, 1700, 3085)])
@pytest.mark.parametrize("xt,yt", [("f32", "f32"), ("bf16", "bf16")])
def test_linear_tiles(hip, M, K, N, xt, yt):
    """Every tile over K of one pair of chunks, several pairs and none, with biases at a cut column edge."""
    test_linear(hip, M, K, N, xt, yt, True)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [(129, 300, 257), (129, 1700, 257), (200, 300, 2570), (2300, 300, 515), (900, 1700, 3085)])
@pytest.mark.parametrize("xt,yt", [("f32", "f32"), ("f16", "f16")])
def test_glu_tiles(hip, M, K, N, xt, yt):
    test_glu(hip, M, K, N, xt, yt, True)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 9, 50, 400])
def test_not_finite(hip, M):
    """A row with an Inf or NaN gives NaN in that row alone; a weight row with byte 255 in that column alone."""
    r = rng(M)
    K, N = 96, 70
    x = randn(r, (M, K))
    x[M // 2, 40] = np.inf
    q, s = mx4.quant(randn(r, (N, K)))
    s[11, 2] = 255
    got = run_linear(hip, "aria_hip_linear_mx4_dev", x, "f32", K, q, s, None, M, K, N, "f32")
    bad = np.zeros((M, N), bool)
    bad[M // 2] = True
    bad[:, 11] = True
    assert np.array_equal(np.isnan(got), bad)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 33, 260])
def test_scale_extremes(hip, M):
    """Block exponents from one end to the other, every scale byte on the weight side too."""
    r = rng(M + 5)
    K, N = 256 * 32, 40
    e = np.arange(256 * 32) // 32 % 256 - 127
    x = (randn(r, (M, K)) * np.ldexp(1.0, np.clip(e, -120, 120))).astype(np.float32)
    q, _ = mx4.quant(randn(r, (N, K)))
    s = np.tile(np.clip(127 - e[::32], 0, 254).astype(np.uint8), (N, 1))
    y, terms = mx4.linear(x, q, s)
    got = run_linear(hip, "aria_hip_linear_mx4_dev", x, "f32", K, q, s, None, M, K, N, "f32")
    assert (np.abs(got - y) <= linear_tol(y, terms, K, "f32")).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [(3, 64, 40), (50, 1000, 129), (700, 512, 256)])
def test_packed_product_is_the_linear(hip, M, K, N):
    """quant_dev + gemm_dev, linear_dev and the host form give the same bits."""
    from aria_amd import ops
    from aria_amd.device import DeviceArray as DA, sync
    r = rng(M)
    x, w, b = randn(r, (M, K)), randn(r, (N, K)), randn(r, N)
    q, s = ops.mx4_quant(w)
    xq, xs = ops.mx4_quant(x)
    a = run_linear(hip, "aria_hip_linear_mx4_dev", x, "f32", K, q, s, b, M, K, N, "f32")
    d = [DA.from_host(v) for v in (xq, xs, q, s, b)]
    dy = DA((M, N))
    hip.check(hip.lib().aria_hip_gemm_mx4_dev(dy.p, 0, d[0].p, d[1].p, d[2].p, d[3].p, d[4].p, M, K, N, None))
    sync()
    y, terms = mx4.linear(x, q, s, b)
    assert (np.abs(dy.to_host() - y) <= linear_tol(y, terms, K, "f32")).all()
    assert np.array_equal(a, ops.linear_mx4(x, q, s, b))
    assert np.array_equal(ops.mx4_dequant(xq, xs, K), mx4.dequant(xq, xs, K).astype(np.float32))


@pytest.mark.gpu
def test_far_rows(hip):
    """Rows of activations more than 2^31 elements apart from the first."""
    from aria_amd.device import DeviceArray as DA, sync
    L = hip.lib()
    r = rng(3)
    M, K, N, ld = 6, 64, 33, (1 << 29) + 8
    x = randn(r, (M, K)).astype(np.float16)
    base = DA(((M - 1) * ld + K) * 2, np.uint8)
    for i in range(M):
        L.aria_cuda_memcpy_h2d(base.p + i * ld * 2, x[i].ctypes.data, K * 2)
    q, s = mx4.quant(randn(r, (N, K)))
    dq, ds, dy, ws = DA.from_host(q), DA.from_host(s), DA((M, N)), DA(int(L.aria_hip_mx4_ws_bytes(M, K)), np.uint8)
    hip.check(L.aria_hip_linear_mx4_dev(dy.p, 0, base.p, 1, ld, dq.p, ds.p, None, M, K, N, ws.p, None))
    sync()
    y, terms = mx4.linear(x.astype(np.float32), q, s)
    assert (np.abs(dy.to_host() - y) <= linear_tol(y, terms, K, "f32")).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [2, 300])
def test_two_streams(hip, M):
    """Two calls at once on streams and workspaces of their own."""
    from aria_amd.device import DeviceArray as DA
    L = hip.lib()
    r = rng(M)
    K, N = 1024, 512
    q, s = mx4.quant(randn(r, (N, K)))
    dq, ds = DA.from_host(q), DA.from_host(s)
    xs = [randn(r, (M, K)) for _ in range(2)]
    dx = [DA.from_host(x) for x in xs]
    dy = [DA((M, N)) for _ in xs]
    ws = [DA(int(L.aria_hip_mx4_ws_bytes(M, K)), np.uint8) for _ in xs]
    st = [L.aria_hip_stream_create() for _ in xs]
    try:
        for _ in range(5):
            for i in range(2):
                hip.check(L.aria_hip_linear_mx4_dev(dy[i].p, 0, dx[i].p, 0, K, dq.p, ds.p, None, M, K, N, ws[i].p, st[i]))
        for i in range(2):
            hip.check(L.aria_hip_stream_sync(st[i]))
    finally:
        for t in st:
            L.aria_hip_stream_destroy(t)
    for i in range(2):
        y, terms = mx4.linear(xs[i], q, s)
        assert (np.abs(dy[i].to_host() - y) <= linear_tol(y, terms, K, "f32")).all()
