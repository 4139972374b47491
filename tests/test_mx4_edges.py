"""MXFP4 at the edges of what its entry points take: row counts, packs, gates. Refusals run on the CPU."""
from __future__ import annotations

import numpy as np
import pytest


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
