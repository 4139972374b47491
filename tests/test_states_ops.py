"""aria_amd.ops on rotary positions, e4m3 rows and attention over shared prefixes: host arrays in and out, and what the
kernels' assembly has to hold."""
from __future__ import annotations

import numpy as np
import pytest

from conftest import randn, rng
from oracle import states
from test_cross_attn import tolerance
from test_mfma_waits import assembly, early_reads, hipcc, parse


def test_shapes_refused():
    from aria_amd import ops
    z = np.zeros
    for bad in (lambda: ops.rotary(z((1, 2, 3, 64)), z((4, 32)), z((4, 16))), lambda: ops.rotary(z((1, 2, 3, 64)), z(32), z(32)),
                lambda: ops.rotary(z((1, 2, 3, 64)), z((4, 32)), z((4, 32)), k=z((1, 3, 3, 64))),
                lambda: ops.rotary(z((1, 2, 3, 64)), z((4, 32)), z((4, 32)), pos=[1, 2]),
                lambda: ops.rotary(z((1, 2, 3, 64)), z((4, 32)), z((4, 32)), first=[1, 2]),
                lambda: ops.e4m3_values(z((4, 16), np.uint8), z(3, np.uint8)),
                lambda: ops.prefix_attention(z((2, 1, 4, 64)), z((1, 5, 2, 64)), z((1, 5, 2, 32))),
                lambda: ops.prefix_attention(z((2, 1, 4, 64)), z((1, 5, 2, 64)), z((1, 5, 2, 64)), z((3, 2, 2, 64)), z((3, 2, 2, 64))),
                lambda: ops.prefix_attention(z((2, 1, 4, 64)), z((1, 5, 2, 64)), z((1, 5, 2, 64)), prefix_len=[1, 2])):
        with pytest.raises(ValueError):
            bad()


@hipcc
def test_inline_asm_behind_mfma(tmp_path):
    """As tests/test_mfma_waits.py has it of the other attention kernels."""
    kernels = parse(assembly(tmp_path, "k_pattn"))
    assert any(op.startswith("v_mfma") for b in kernels.values() for _, ins in b for _, op, _, _ in ins)
    bad = {name: r[:3] for name, b in kernels.items() if (r := early_reads(b))}
    assert not bad, bad


@pytest.mark.gpu
def test_rotary(hip):
    from aria_amd import ops
    r = rng(1)
    cos, sin = ops.rotary_tables(40, 32, first=3, scaling="linear", factor=4.0)
    want = states.table(32, 3, 40, kind=1, factor=4.0)
    assert max(np.abs(cos - want[0]).max(), np.abs(sin - want[1]).max()) <= 2.0 ** -22
    q, k = randn(r, (2, 9, 4, 64)), randn(r, (2, 9, 2, 64))
    pos = r.integers(0, 40, (2, 9))
    pos[0, 3] = -1
    got = ops.rotary(q, cos, sin, k=k, pos=pos, interleaved=True)
    for x, y in zip((q, k), got):
        want, _ = states.rotate(x, cos[pos][:, :, None], sin[pos][:, :, None], True)
        want[0, 3] = x[0, 3]
        assert np.abs(y - want).max() <= 2.0 ** -24 * np.abs(want).max()
    again = ops.rotary(got[0], cos, sin, pos=pos, interleaved=True, inverse=True)
    assert np.abs(again - q).max() <= 8 * 2.0 ** -23 * np.abs(q).max()


@pytest.mark.gpu
def test_far_positions_are_outside(hip):
    """A position of 2^32 or -2^40 is outside the table like any other, and does not come back into it as 32 bits."""
    from aria_amd import ops
    cos, sin = ops.rotary_tables(8, 32)
    q = randn(rng(4), (3, 2, 4, 64))
    pos = np.array([[2 ** 32 + 5, 3], [-2 ** 40, 2 ** 63 - 1], [7, 2 ** 31]])
    got = ops.rotary(q, cos, sin, pos=pos)
    want = q.copy()
    for b, t in ((0, 1), (2, 0)):
        want[b, t], _ = states.rotate(q[b, t], cos[pos[b, t]], sin[pos[b, t]], False)
    assert np.abs(got - want).max() <= 2.0 ** -24 * np.abs(want).max()
    got = ops.rotary(q, cos, sin, first=[2 ** 32, -2 ** 32, 6])
    want = q.copy()
    for t in (0, 1):
        want[2, t], _ = states.rotate(q[2, t], cos[6 + t], sin[6 + t], False)
    assert np.abs(got - want).max() <= 2.0 ** -24 * np.abs(want).max()


@pytest.mark.gpu
def test_nothing_to_do(hip):
    from aria_amd import ops
    z = np.zeros
    cos, sin = ops.rotary_tables(0, 32)
    assert cos.shape == sin.shape == (0, 16)
    assert ops.rotary(z((2, 0, 4, 64)), z((4, 16)), z((4, 16))).shape == (2, 0, 4, 64)
    x = randn(rng(5), (1, 3, 4, 64))
    assert np.array_equal(ops.rotary(x, cos, sin), x), "every position is outside an empty table"
    code, byte = ops.e4m3_rows(z((0, 32)))
    assert code.shape == (0, 32) and byte.shape == (0,) and ops.e4m3_values(code, byte).shape == (0, 32)
    assert ops.prefix_attention(z((2, 0, 4, 64)), z((1, 5, 2, 64)), z((1, 5, 2, 64))).shape == (2, 0, 4, 64)
    assert not ops.prefix_attention(x, z((1, 0, 2, 64)), z((1, 0, 2, 64))).any(), "rows that see no key are zero"


@pytest.mark.gpu
def test_rows(hip):
    import aria_amd
    from aria_amd import ops
    x = randn(rng(2), (3, 5, 48)) * 7
    x[1, 2] = 0
    code, byte = ops.e4m3_rows(x)
    assert all(np.array_equal(a, b) for a, b in zip((code, byte), states.rows(x)))
    assert np.array_equal(ops.e4m3_values(code, byte), states.values(code, byte))
    with pytest.raises(aria_amd.HipError):
        ops.e4m3_rows(x[..., :40])


@pytest.mark.gpu
@pytest.mark.parametrize("m", [0, 12])
def test_prefix_attention(hip, m):
    from aria_amd import ops
    r = rng(3)
    B, Nq, H, Hkv, D, P, n = 4, 3, 4, 2, 64, 2, 50
    q = randn(r, (B, Nq, H, D)).astype(np.float16).astype(np.float32)
    pk, pv, k, v = (randn(r, s) for s in ((P, n, Hkv, D),) * 2 + ((B, m, Hkv, D),) * 2)
    pl, ol, first = [n, 2 ** 40], [m, 0, m // 2, m], [m - Nq] * B
    got = ops.prefix_attention(q, pk, pv, k if m else None, v if m else None, prefix_len=pl, own_len=ol, first=first)
    cached = [states.values(*states.rows(x)).transpose(0, 2, 1, 3) for x in (pk, pv, k, v)]
    qt = q.transpose(0, 2, 1, 3)
    want, mag = states.attention(qt, cached[:2], cached[2:], [n, n], ol, first)
    kk, vv = (np.concatenate((cached[i].ravel(), cached[2 + i].ravel())) for i in range(2))
    assert (np.abs(got - want) <= tolerance(want, mag, qt, kk, vv, "f16", "f32", 1 / np.sqrt(D), n + m)).all()
