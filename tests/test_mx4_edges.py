"""MXFP4 at the edges of what its entry points take: row counts, packs, gates. Refusals run on the CPU."""
from __future__ import annotations

import numpy as np
import pytest

from conftest import randn, rng
from oracle import mx4
from test_mx4 import run_linear


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
