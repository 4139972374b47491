"""The scale bytes and codes of rotated rows whose width leaves lanes of the kernel's groups without a chunk of their own: to the
bit, against the definition in 64 bits (oracle/states.py)."""
from __future__ import annotations

import numpy as np
import pytest

import test_states as ts
from conftest import randn, rng
from oracle import states

WIDTHS = (16, 48, 80, 96, 112, 144, 160, 176, 208, 240)


def write(hip, x, t, cos, sin, inter):
    """x [N, heads, D] as keys and as values of one sequence, keys rotated by the tables' rows -> [(codes, bytes), ...]"""
    from aria_amd.device import sync
    N, h, D = x.shape
    k, kv = ts.cast(x[None], t)
    lk, c = ts.Laid(k), ts.Cache(hip, 1, h, N, D)
    dc, ds = ts.dev(cos, np.float32), ts.dev(sin, np.float32)
    w = hip.KVWrite(cache=c.c, k=lk.p, v=lk.p, cos=dc.p, sin=ds.p, type=ts.CODE[t], N=N, rot=2 * cos.shape[1], npos=len(cos), interleaved=inter)
    ts.strides(w, "k", lk)
    ts.strides(w, "v", lk)
    hip.check(hip.lib().aria_hip_kv_write_dev(w, None))
    sync()
    y, _ = states.rotate(kv[0], cos[:, None], sin[:, None], inter)
    return [c.get(i) for i in range(2)], [states.rows(y.astype(np.float32)), states.rows(kv[0])]


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("D", WIDTHS)
def test_rotated_rows(hip, t, inter, D):
    """Prompts and single tokens, with queries beside them, read back in every type."""
    ts.test_write_and_read(hip, t, inter, 2, 150, 3, D, D, "tokens", 3, 2)
    ts.test_write_and_read(hip, t, inter, 5, 1, 2, D, D, "heads", 0, 4)


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("D,rot", [(D, D) for D in WIDTHS + (32, 64, 128, 256)] + [(80, 64), (96, 48), (112, 96), (80, 20)])
def test_largest_before_the_rotation(hip, t, inter, D, rot):
    """One large number at each dim in turn, turned by an eighth: the row's largest is smaller by sqrt(1/2) afterwards, which
    crosses a power of two. What the row held before the rotation does not count."""
    r = rng(D + rot)
    x = np.clip(randn(r, (D, 2, D)), -3, 3) * 2.0 ** -11
    x[np.arange(D), :, np.arange(D)] = 2.0
    eighth = np.full((D, rot // 2), np.sqrt(0.5), np.float32)
    got, want = write(hip, x, t, eighth, eighth, inter)
    assert set(np.unique(want[0][1])) == ({119, 120} if rot < D else {119})
    for i in range(2):
        assert np.array_equal(got[i][1][0], want[i][1]), "bytes of " + "kv"[i]
        assert np.array_equal(got[i][0][0], want[i][0]), "codes of " + "kv"[i]


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("D", [16, 48, 80, 96])
def test_many_rows(hip, t, inter, D):
    """Normal states of many tokens at their positions."""
    N = 700
    cos, sin = ts.some_table(D, N)
    got, want = write(hip, randn(rng(D), (N, 4, D)), t, cos, sin, inter)
    for i in range(2):
        assert np.array_equal(got[i][1][0], want[i][1]) and np.array_equal(got[i][0][0], want[i][0])
