"""Rotary tables of pairs that turn fast, at far positions: as precise as any, or refused (oracle/states.py)."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import states

P = 4096     # never dereferenced


def scaling(**kw):
    import aria_amd
    return aria_amd.RotaryScaling(**(dict(rot=64, kind=0, base=10000.0, factor=1.0, trained=1.0, low=1.0, high=2.0, gain=1.0) | kw))


# ---- CPU ----

def test_more_than_16_turns_a_position():
    import aria_amd
    for kw in (dict(kind=1, factor=1e-6), dict(kind=1, factor=0.0099), dict(kind=3, factor=1e-6), dict(kind=2, factor=1e-6)):
        assert aria_amd.lib().aria_hip_rotary_table_dev(P, P, scaling(**kw), 0, 4, None) == -1, kw
        assert "invalid argument" in aria_amd.last_error()
    assert aria_amd.lib().aria_hip_rotary_table_dev(P, P, scaling(kind=1, factor=0.01), 0, 0, None) == 0


@pytest.mark.parametrize("gain", [1e39, -3.5e38, 1e300])
def test_gain_beyond_fp32(gain):
    """It would be infinite in the tables' type, and 0 times it not a number."""
    import aria_amd
    assert aria_amd.lib().aria_hip_rotary_table_dev(P, P, scaling(gain=gain), 0, 4, None) == -1
    assert "invalid argument" in aria_amd.last_error()
    assert aria_amd.lib().aria_hip_rotary_table_dev(P, P, scaling(gain=gain * 1e-300), 0, 0, None) == 0


# ---- GPU ----

@pytest.mark.gpu
@pytest.mark.parametrize("first", [0, (1 << 24) - 299])
@pytest.mark.parametrize("kw", [dict(), dict(kind=1, factor=0.5), dict(kind=1, factor=0.02), dict(kind=1, factor=0.01),
                                dict(kind=3, factor=0.0103), dict(kind=2, factor=1e-5), dict(kind=1, factor=1 / 3, rot=250)])
def test_fast_pairs(hip, first, kw):
    """The reduced turns are known to 2^-55 and, before they are reduced, to 128 steps of 2^-64 of 16 turns; with a position of 2^24 and the product's
    own half step that is 2^-31 + 2^-29 + 2^-31 turns, below 2^-28. What is left of them as an fp32 number of an eighth of a turn at most: 2^-28 more. 2 pi
    times both; the series behind them and their roundings within 2^-23 of 1."""
    from aria_amd.device import DeviceArray as DA, sync
    a = scaling(**kw)
    n = 300
    d = [DA((n, a.rot // 2)) for _ in range(2)]
    hip.check(hip.lib().aria_hip_rotary_table_dev(d[0].p, d[1].p, a, first, n, None))
    sync()
    want = states.table(a.rot, first, n, kind=a.kind, factor=a.factor, trained=1.0, low=1.0, high=2.0)
    for x, y in zip(d, want):
        assert np.abs(x.to_host() - y).max() <= 2 * np.pi * 2.0 ** -27 + 2.0 ** -23


@pytest.mark.gpu
@pytest.mark.parametrize("rot,n", [(128, 40961), (38, 5003), (256, 9000), (6, 100000)])
def test_many_positions(hip, rot, n):
    """Every position of a grid of many workgroups, whole groups of pairs and single ones."""
    from aria_amd.device import DeviceArray as DA, sync
    first = 1000003
    d = [DA.from_host(np.full((n + 1, rot // 2), 99, np.float32)) for _ in range(2)]
    hip.check(hip.lib().aria_hip_rotary_table_dev(d[0].p, d[1].p, scaling(rot=rot), first, n, None))
    sync()
    for x, y in zip(d, states.table(rot, first, n)):
        x = x.to_host()
        assert (x[n] == 99).all() and np.abs(x[:n] - y).max() <= 2 * np.pi * 2.0 ** -27 + 2.0 ** -23
