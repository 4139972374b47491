"""MXFP4 at the edges of what its entry points take: row counts, packs, gates. Refusals run on the CPU."""
from __future__ import annotations

import numpy as np
import pytest

from conftest import randn, rng
from oracle import mx4
from test_mx4 import CODE, cast, np_type, run_linear, values


# ---- CPU ----

@pytest.mark.parametrize("rows", [(1 << 30) + 1, 2147483137, (1 << 31) - 1])
def test_row_counts_refused(rows):
    """More rows than the launches' arithmetic holds (2147483137 is the first at which rows taken in launches of
    268435392 pass 2^31): refused before any device work, with pointers that are never dereferenced."""
    import aria_amd
    L = aria_amd.lib()
    p = 4096

    def bad(rc, what):
        assert rc == -1, rc
        assert what in aria_amd.last_error(), aria_amd.last_error()
    bad(L.aria_hip_mx4_quant_dev(p, p, p, 1, rows, 1, 1, None), "rows <=")
    bad(L.aria_hip_mx4_dequant_dev(p, 1, p, p, rows, 1, None), "rows <=")
    bad(L.aria_hip_mx4_quant(p, p, p, rows, 1), "rows <=")
    bad(L.aria_hip_mx4_dequant(p, p, p, rows, 1), "rows <=")


@pytest.mark.parametrize("M,N", [((1 << 28) + 1, 1), ((1 << 31) - 1, 1), (5 * 10 ** 8 + 4 * 10 ** 7, 32),
                                 (1 << 20, (1 << 16) + 1), ((1 << 10) + 1, 1 << 26)])
def test_products_refused(M, N):
    """More rows than 2^28 or more outputs than 2^36, the gated form included."""
    import aria_amd
    L = aria_amd.lib()
    p = 4096
    for fn in (L.aria_hip_linear_mx4_dev, L.aria_hip_glu_mx4_dev):
        assert fn(p, 1, p, 1, 32, p, p, None, M, 32, N, p, None) == -1
        assert "MX4_FITS" in aria_amd.last_error()
    assert L.aria_hip_gemm_mx4_dev(p, 1, p, p, p, p, None, M, 32, N, None) == -1 and "MX4_FITS" in aria_amd.last_error()
    for fn in (L.aria_hip_linear_mx4, L.aria_hip_glu_mx4):
        assert fn(p, p, p, p, None, M, 32, N) == -1 and "MX4_FITS" in aria_amd.last_error()


@pytest.mark.parametrize("shape", [(3,), (5,), (1,), (0,), (2, 4), ()])
def test_bias_of_another_size(shape):
    """The numpy forms read one bias per weight row: another number of them is refused, not read past its end."""
    from aria_amd import ops
    x, q, s = np.zeros((2, 32), np.float32), np.zeros((4, 16), np.uint8), np.zeros((4, 1), np.uint8)
    for fn in (ops.linear_mx4, ops.glu_mx4):
        with pytest.raises(ValueError, match="bias"):
            fn(x, q, s, np.zeros(shape, np.float32))


# ---- GPU ----

@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 40, 300, 1300])
def test_gate_far_from_zero(hip, M):
    """SiLU of gates from -85 to 85 in fp32. Products are zero, so the gates are the biases, exactly, and the values 1:
    exp2 and rcp are a step (two half steps) each, the factor and the four products and sums half a step each: 9 half steps, whatever
    the gate."""
    r = rng(M)
    K, N = 96, 2050
    q, s = mx4.quant(randn(r, (2 * N, K)))
    b = np.concatenate([np.ones(N), np.linspace(-85, 85, N)]).astype(np.float32)
    got = run_linear(hip, "aria_hip_glu_mx4_dev", np.zeros((M, K), np.float32), "f32", K, q, s, b, M, K, N, "f32")
    g = b[N:].astype(np.float64)
    want = g / (1 + np.exp(-g))
    assert (np.abs(got - want) <= 9.01 * 2.0 ** -24 * np.abs(want)).all(), (np.abs(got - want) / np.abs(want)).max() * 2 ** 24


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 200])
def test_gate_limits(hip, M):
    """Gates past e^-g's range: v g above, nothing below; an infinite gate gives v times infinity, or NaN as -Inf / Inf does."""
    K = 32
    gates = np.array([88.0, 104.5, 3e38, np.inf, -104.5, -3e38, -np.inf, np.nan, 0.0], np.float32)
    N = len(gates)
    q, s = mx4.quant(np.zeros((2 * N, K)))
    b = np.concatenate([np.full(N, 0.5, np.float32), gates])
    got = run_linear(hip, "aria_hip_glu_mx4_dev", np.zeros((M, K), np.float32), "f32", K, q, s, b, M, K, N, "f32")
    want = np.array([44.0, 52.25, 1.5e38, np.inf, 0, 0, np.nan, np.nan, 0])
    assert np.allclose(got, want[None], rtol=2.0 ** -21, atol=0, equal_nan=True)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [(700, 512, 256), (17, 2048, 96), (344, 4096, 1024), (2592, 1024, 1030)])
@pytest.mark.parametrize("xt,yt,bias", [("f32", "f32", True), ("bf16", "f16", False)])
def test_quantised_apart_gives_the_same_bits(hip, M, K, N, xt, yt, bias):
    """Where the linear takes two launches, quantising first and multiplying the packed operands is the same to the bit."""
    from aria_amd.device import DeviceArray as DA, sync
    L = hip.lib()
    r = rng(M + N)
    x, _ = cast(randn(r, (M, K)), xt)
    q, s = mx4.quant(randn(r, (N, K)))
    b = randn(r, N) if bias else None
    want = run_linear(hip, "aria_hip_linear_mx4_dev", x, xt, K, q, s, b, M, K, N, yt)
    dx, dq, ds = DA.from_host(x), DA.from_host(q), DA.from_host(s)
    db = DA.from_host(b) if bias else None
    xq, xs, dy = DA((M, K // 2), np.uint8), DA((M, K // 32), np.uint8), DA((M, N), np_type(yt))
    hip.check(L.aria_hip_mx4_quant_dev(xq.p, xs.p, dx.p, CODE[xt], M, K, K, None))
    hip.check(L.aria_hip_gemm_mx4_dev(dy.p, CODE[yt], xq.p, xs.p, dq.p, ds.p, db.p if bias else None, M, K, N, None))
    sync()
    assert np.array_equal(values(dy.to_host(), yt), want)


@pytest.mark.gpu
def test_rows_of_several_launches(hip):
    """More rows than one launch of the quantiser takes (268435392 at K up to 32): the border between two launches, both
    ends, and what lies behind the last row."""
    from aria_amd.device import DeviceArray as DA, sync
    L = hip.lib()
    border, period = 268435392, 4096
    rows = border + 70001
    x = np.resize(np.ldexp(randn(rng(1), period), np.arange(period) % 20 - 10).astype(np.float16), rows)
    want_q, want_s = mx4.quant(x[:period, None].astype(np.float32))
    dx, dq, ds = DA.from_host(x), DA((rows + 8, 16), np.uint8), DA(rows + 8, np.uint8)
    fill = np.full(128, 0xAB, np.uint8)
    L.aria_cuda_memcpy_h2d(dq.p + 16 * rows, fill.ctypes.data, 128)
    L.aria_cuda_memcpy_h2d(ds.p + rows, fill.ctypes.data, 8)
    print(f"[gpu] mx4 quant rows {rows}", flush=True)
    hip.check(L.aria_hip_mx4_quant_dev(dq.p, ds.p, dx.p, CODE["f16"], rows, 1, 1, None))
    dy = DA(rows + 8, np.float16)
    L.aria_cuda_memcpy_h2d(dy.p + 2 * rows, fill.ctypes.data, 16)
    hip.check(L.aria_hip_mx4_dequant_dev(dy.p, CODE["f16"], dq.p, ds.p, rows, 1, None))
    sync()

    def part(d, first, n, size, dtype):
        out = np.empty((n, size // np.dtype(dtype).itemsize), dtype)
        L.aria_cuda_memcpy_d2h(out.ctypes.data, d.p + first * size, n * size)
        return out
    v = mx4.dequant(want_q, want_s, 1).astype(np.float16)
    for first, n in ((0, 5000), (border - 5000, 10000), (rows - 5000, 5000)):
        at = np.arange(first, first + n) % period
        assert np.array_equal(part(dq, first, n, 16, np.uint8), want_q[at])
        assert np.array_equal(part(ds, first, n, 1, np.uint8), want_s[at])
        assert np.array_equal(part(dy, first, n, 2, np.float16), v[at])
    assert (part(dq, rows, 8, 16, np.uint8) == 0xAB).all() and (part(ds, rows, 8, 1, np.uint8) == 0xAB).all()
    assert (part(dy, rows, 8, 2, np.uint16) == 0xABAB).all()
