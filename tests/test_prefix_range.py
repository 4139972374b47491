"""Attention over cached keys and values that lie beyond the query type's range: they are held to it, as reading the cache does,
and rows that do not see them are untouched (oracle/states.py)."""
from __future__ import annotations

import numpy as np
import pytest

from conftest import randn, rng
from oracle import states
from test_cross_attn import tolerance
from test_prefix_attn import fill, run
from test_states import LARGEST, cast

# B, prefixes, H, Hkv, Nq, prefix, own, D: every form, rows of a prefix together and alone, joined and not, widths beside a product's
SHAPES = [(1, 1, 1, 1, 1, 20, 5, 64), (8, 1, 4, 1, 1, 700, 90, 128), (2, 1, 4, 2, 20, 40, 40, 48), (3, 3, 4, 2, 24, 33, 70, 128),
          (2, 1, 4, 4, 150, 70, 160, 64), (2, 2, 2, 1, 70, 0, 130, 112), (2, 1, 8, 8, 140, 100, 140, 80), (4, 2, 2, 2, 33, 3000, 40, 32)]


def place(c, which, b, slot, dim, big):
    """Row `slot` of the first key head of b: its values with `big` among them, as the cache holds them -> what was there"""
    code, byte = c.get(which)
    old = code.copy(), byte.copy()
    code, byte = code.copy(), byte.copy()
    x = states.values(code[b, slot, 0], byte[b, slot, 0])
    x[dim] = big
    code[b, slot, 0], byte[b, slot, 0] = states.rows(x[None])[0][0], states.rows(x[None])[1][0]
    c.put(which, code, byte)
    return old, states.values(code, byte).transpose(0, 2, 1, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("t,big", [("f16", 65504.0), ("f16", -65504.0), ("f16", 1e6), ("f16", -3e38), ("bf16", 3.3895313892515355e38),
                                   ("bf16", -3.4028e38)])
@pytest.mark.parametrize("shape", SHAPES)
def test_beyond_the_type(hip, t, big, shape):
    B, Pn, H, Hkv, Nq, n, m, D = shape
    r, G, dim, top = rng(sum(shape)), H // Hkv, D - 3, LARGEST[t]
    print(f"[gpu] prefix attention {t}, {big} among {shape}", flush=True)
    q = randn(r, (B, H, Nq, D))
    q[..., dim] = 0                          # so that a large key's score stays that of the others
    q, qv = cast(q, t)
    cp, pv = fill(hip, r, Pn, Hkv, n, D)
    co, ov = fill(hip, r, B, Hkv, m, D)
    first = np.full(B, m - Nq)
    clean = run(hip, t, q, cp, co, first=first, out="f32")
    slot = m - 1 - Nq // 2
    for c, at, own in ((co, slot, True), (cp, n // 2, False)):
        if not own and n == 0:
            continue
        seen = np.zeros((B, Nq, H), bool)
        if own:
            seen[0, :, :G] = (first[0] + np.arange(Nq) >= slot)[:, None]
        else:
            seen[:B // Pn, :, :G] = True
        for which in (0, 1):
            old, val = place(c, which, 0, at, dim, big)
            got = run(hip, t, q, cp, co, first=first, out="f32")
            c.put(which, *old)
            assert np.array_equal(got[~seen], clean[~seen]), "a row that does not see it"
            if t == "bf16" and which == 1:   # its product with a weight of 2^7 and more is beyond fp32
                assert not np.isnan(got).any()
                continue
            pk, ok = [list(x) for x in (pv, ov)]
            (ok if own else pk)[which] = np.clip(val, -top, top)
            want, mag = states.attention(qv, pk, ok, None, None, first)
            k, v = (np.concatenate((pk[i].ravel(), ok[i].ravel())) for i in range(2))
            tol = tolerance(want, mag, qv, np.where(np.abs(k) < 1e3, k, 0.0), v, t, "f32", 1 / np.sqrt(D), n + m)
            assert np.isfinite(got).all() and (np.abs(got - want) <= tol).all(), np.nanmax(np.abs(got - want) - tol)


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("B,Nq,m,D", [(1, 8, 40, 64), (3, 40, 90, 128), (2, 150, 170, 96)])
def test_beside_a_row_that_is_nan(hip, t, B, Nq, m, D):
    """A large value, a row of byte 255 and a large key in one tile, slot by slot: each reaches the rows behind it alone."""
    r = rng(Nq)
    q = randn(r, (B, 2, Nq, D))
    q[..., D - 3] = 0
    q, _ = cast(q, t)
    cp, co = fill(hip, r, 1, 1, 20, D)[0], fill(hip, r, B, 1, m, D)[0]
    first, slot = np.full(B, m - Nq), m - Nq // 2
    clean = run(hip, t, q, cp, co, first=first, out="f32")
    place(co, 1, 0, slot, D - 3, 0.25 * LARGEST[t] if t == "bf16" else 2.0 * LARGEST[t])
    for i in range(2):
        code, byte = (x.copy() for x in co.get(i))
        code[0, slot + 1], byte[0, slot + 1] = 0x7F, 255
        co.put(i, code, byte)
    place(co, 0, 0, slot + 2, D - 3, -LARGEST[t])
    got = run(hip, t, q, cp, co, first=first, out="f32")
    last = first[0] + np.arange(Nq)          # the last slot that a token sees
    assert np.array_equal(got[1:], clean[1:]) and np.array_equal(got[0, last < slot], clean[0, last < slot])
    assert not np.isnan(got[0, last == slot]).any() and np.isnan(got[0, last > slot]).all()


@pytest.mark.gpu
def test_finite_states_stay_finite(hip):
    """Host arrays whose values fp16 does not reach."""
    from aria_amd import ops
    r = rng(5)
    q, pk, pv = randn(r, (2, 3, 4, 64)).astype(np.float16).astype(np.float32), *(randn(r, (1, 50, 2, 64)) for _ in range(2))
    pv[0, 7] *= 1e5
    held = [states.values(*states.rows(x)).transpose(0, 2, 1, 3) for x in (pk, pv)]
    held[1] = np.clip(held[1], -65504.0, 65504.0)
    got = ops.prefix_attention(q, pk, pv)
    qt = q.transpose(0, 2, 1, 3)
    none = [np.zeros((2, 2, 0, 64))] * 2
    want, mag = states.attention(qt, held, none)
    assert (np.abs(got - want) <= tolerance(want, mag, qt, held[0], held[1], "f16", "f32", 1 / 8, 50)).all()
