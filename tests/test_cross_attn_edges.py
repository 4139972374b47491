"""Cross attention where values, scores or descriptions lie at an edge, against the definition in 64 bits
(oracle/mx4.py). Refusals run on the CPU."""
from __future__ import annotations

import numpy as np
import pytest

from conftest import randn, rng
from oracle import mx4
from test_cross_attn import cast, describe, run, tolerance

# every form of workgroup: four slices of one wave (split over workgroups too), four waves and two slices, four waves, eight
FORMS = [(1, 8, 2, 3, 700, 64), (1, 4, 4, 5, 700, 128), (1, 16, 8, 1100, 600, 64), (2, 8, 8, 1025, 300, 128), (3, 16, 16, 1000, 300, 64),
         (3, 16, 16, 1000, 200, 72), (8, 16, 16, 2050, 100, 64)]


# ---- CPU ----

def test_workspace_before_the_pointers():
    """The workspace of a call goes by its sizes: a description without pointers, strides, type or scale gives the same
    number, and not the 0 that says that there is none."""
    import aria_amd
    L = aria_amd.lib()
    sizes = dict(B=16, H=16, Hkv=4, Nq=1, Nk=8192, D=128)
    full = describe(aria_amd, "bf16", *sizes.values())
    full.q = full.k = full.v = full.out = 4096
    want = L.aria_hip_cross_attention_ws_bytes(full)
    assert want > 0
    assert L.aria_hip_cross_attention_ws_bytes(aria_amd.CrossAttention(**sizes)) == want
    assert L.aria_hip_cross_attention_ws_bytes(aria_amd.CrossAttention(**{**sizes, "D": 12})) == 0
    bare = aria_amd.CrossAttention(**sizes)
    assert L.aria_hip_cross_attention_dev(bare, 4096, None) == -1       # still refused as a call


@pytest.mark.parametrize("scale,taken", [(2.0 ** 127, True), (2.0 ** 127 * 1.0625, False), (3.4e38, False)])
def test_largest_scale(scale, taken):
    """Scores are taken times scale log2 e, which has to be finite itself: a score of 0 would be NaN. (No rows: a call that
    is taken has nothing to do.)"""
    import aria_amd
    a = describe(aria_amd, "bf16", 1, 1, 1, 0, 8, 64, scale)
    assert aria_amd.lib().aria_hip_cross_attention_dev(a, None, None) == (0 if taken else -1)


@pytest.mark.parametrize("lens,want", [([2 ** 32, 2 ** 32 + 3], [5, 5]), ([-2 ** 40, 2], [0, 2]), ([3.0, 1e12], [3, 5])])
def test_lengths_of_other_types(monkeypatch, lens, want):
    """Lengths past 32 bits are clamped to 0..Nk like any other, not cut off to their low bits."""
    import ctypes
    from aria_amd import ops
    seen = []

    class Lib:
        def aria_hip_cross_attention_f16(self, out, q, k, v, kv_len, mask, *sizes):
            seen.extend(ctypes.cast(kv_len, ctypes.POINTER(ctypes.c_int32))[:2])
            return 0
    monkeypatch.setattr(ops, "lib", Lib)
    z = np.zeros((2, 1, 5, 64), np.float32)
    ops.cross_attention(z, z, z, kv_len=lens)
    assert seen == want


# ---- GPU ----

@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("B,H,Hkv,Nq,Nk,D", FORMS)
def test_masked_keys_above_low_scores(hip, t, B, H, Hkv, Nq, Nk, D):
    """Every valid score is -60 or less, a masked key's products alone would be 0: a maximum that saw those would leave no
    weight in 16 bits."""
    print(f"[gpu] low scores {t} {B} {H}/{Hkv} {Nq} {Nk} {D}", flush=True)
    r = rng(Nq + Nk)
    q, qv = cast(1.0 + 0.05 * randn(r, (B, H, Nq, D)), t)
    k, kv = cast(-90.0 / np.sqrt(D) + 0.05 * randn(r, (B, Hkv, Nk, D)), t)
    v, vv = cast(randn(r, (B, Hkv, Nk, D)), t)
    mask = (r.random((B, Nk)) < 0.4).astype(np.uint8)
    got = run(hip, t, q, k, v, mask=mask)
    want, mag = mx4.cross_attention(qv, kv, vv, mask=mask)
    assert qv.min() > 0 and qv.min() * kv.max() * np.sqrt(D) < -60
    assert (np.abs(got - want) <= tolerance(want, mag, qv, kv, vv, t, t, 1 / np.sqrt(D), Nk)).all(), np.abs(got - want).max()


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Hkv,Nq,Nk,D", FORMS)
def test_many_small_weights(hip, B, H, Hkv, Nq, Nk, D):
    """fp16: one key of weight 1 and value 0, all others of weight 2^-25.1 and large values, which make the whole
    result. A weight is held to half a step of fp16's smallest numbers, 2^-25, against a largest weight of at least 2^6.5
    (2^7 less the reference's rounding): 2^-31.5 of the largest."""
    print(f"[gpu] small weights {B} {H}/{Hkv} {Nq} {Nk} {D}", flush=True)
    r = rng(Nk)
    q, qv = cast(np.ones((B, H, Nq, D), np.float32), "f16")
    kf = np.full((B, Hkv, Nk, D), -17.4 / np.sqrt(D), np.float32)
    kf[:, :, Nk // 2] = 0
    vf = 2000.0 + 100 * randn(r, (B, Hkv, Nk, D))
    vf[:, :, Nk // 2] = 0
    (k, kv), (v, vv) = cast(kf, "f16"), cast(vf, "f16")
    got = run(hip, "f16", q, k, v, out="f32")
    want, mag = mx4.cross_attention(qv, kv, vv)
    assert (np.abs(want) > 1e-3).all()
    tol = Nk * 2.0 ** -31.5 * vv.max() + tolerance(want, mag, qv, kv, 0 * vv, "f16", "f32", 1 / np.sqrt(D), 0)
    assert (tol < 0.1 * want).all()
    assert (np.abs(got - want) <= tol).all(), (got.min(), want.min())


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("B,H,Hkv,Nq,Nk,D", FORMS)
def test_far_scores(hip, t, sign, B, H, Hkv, Nq, Nk, D):
    """Scores so large that fp32's steps are 64: q and k are such that every score is exact, so a row's weights are those of
    its largest keys alone, equal where they tie."""
    print(f"[gpu] far scores {t} {sign} {B} {H}/{Hkv} {Nq} {Nk} {D}", flush=True)
    r = rng(Nq + Nk)
    q = np.zeros((B, H, Nq, D), np.float32)
    k = np.zeros((B, Hkv, Nk, D), np.float32)
    q[..., 0] = 32768
    k[..., 0] = sign * 128 * r.integers(248, 256, (B, Hkv, Nk))   # scores just under 2^30 in size, whole multiples of 64, fp32's step
    q[..., 1] = 8 * r.integers(0, 2, (B, H, Nq))                  # there; in half of the rows the largest are a few steps apart
    k[..., 1] = 8 * r.integers(0, 4, (B, Hkv, Nk))
    (q, qv), (k, kv), (v, vv) = cast(q, t), cast(k, t), cast(randn(r, (B, Hkv, Nk, D)), t)
    got = run(hip, t, q, k, v, out="f32", scale=1.0)
    want, mag = mx4.cross_attention(qv, kv, vv, scale=1.0)
    # the weights are 1 / ties of each row, exact before the sum's rounding and the division
    tol = (Nk + 8) * 2.0 ** -23 * (mag + np.abs(want))
    assert (np.abs(got - want) <= tol).all(), np.abs(got - want).max()
    lens, mask = r.integers(0, Nk + 1, B), (r.random((B, Nk)) < 0.5).astype(np.uint8)
    got = run(hip, t, q, k, v, lens, mask, out="f32", layout="tokens", scale=1.0)
    want, mag = mx4.cross_attention(qv, kv, vv, lens, mask, scale=1.0)
    assert (np.abs(got - want) <= (Nk + 8) * 2.0 ** -23 * (mag + np.abs(want))).all()


@pytest.mark.gpu
@pytest.mark.parametrize("Nq", [1, 200])
def test_lowest_scores(hip, Nq):
    """bf16: every score -1.375 x 2^127, which in base 2 is just inside fp32: the mean of the values, not a row without weight."""
    r = rng(Nq)
    q, k = np.zeros((1, 2, Nq, 64), np.float32), np.zeros((1, 2, 300, 64), np.float32)
    q[..., 3], k[..., 3] = -2.0 ** 63, 1.375 * 2.0 ** 64
    (q, _), (k, _), (v, vv) = cast(q, "bf16"), cast(k, "bf16"), cast(randn(r, (1, 2, 300, 64)), "bf16")
    got = run(hip, "bf16", q, k, v, out="f32", scale=1.0)
    want = np.broadcast_to(vv.astype(np.float64).mean(2)[:, None], (1, Nq, 2, 64))
    assert (np.abs(got - want) <= 308 * 2.0 ** -23 * np.abs(vv).max()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("B,H,Hkv,Nq,Nk,D", [(2, 4, 2, 1, 200, 64), (2, 4, 2, 3, 900, 128), (2, 4, 2, 300, 200, 64), (2, 8, 4, 1000, 300, 72)])
def test_not_finite(hip, t, B, H, Hkv, Nq, Nk, D):
    """Inf and NaN in queries, valid keys and values go where the definition takes them, and change no bit elsewhere."""
    print(f"[gpu] not finite {t} {Nq} {Nk} {D}", flush=True)
    r = rng(Nq + D)
    G = H // Hkv
    qf, kf, vf = randn(r, (B, H, Nq, D)), randn(r, (B, Hkv, Nk, D)), randn(r, (B, Hkv, Nk, D))
    plain = run(hip, t, cast(qf, t)[0], cast(kf, t)[0], cast(vf, t)[0], out="f32")

    def check(q, k, v, touched):
        with np.errstate(invalid="ignore"):
            (q, qv), (k, kv), (v, vv) = bits(q, t), bits(k, t), bits(v, t)
            got = run(hip, t, q, k, v, out="f32")
            want, mag = mx4.cross_attention(qv, kv, vv)
        same = np.ones(got.shape, bool)
        same[touched] = False
        assert np.array_equal(got[same], plain[same])
        assert np.array_equal(np.isnan(got), np.isnan(want))
        assert np.array_equal(np.isposinf(got), np.isposinf(want)) and np.array_equal(np.isneginf(got), np.isneginf(want))
        ok = np.isfinite(want)
        clean = [np.where(np.isfinite(x), x, 0) for x in (qv, kv, vv)]
        tol = tolerance(want, np.where(np.isfinite(mag), mag, 0), *clean, t, "f32", 1 / np.sqrt(D), Nk)
        assert (np.abs(got[ok] - want[ok]) <= tol[ok]).all()

    h, j, d = H - 1, Nk - 3, 5
    for bad in (np.nan, np.inf, -np.inf):
        q = qf.copy()
        q[0, h, Nq // 2, d] = bad
        check(q, kf, vf, np.s_[0, Nq // 2, h])              # one row, NaN: some of its scores are +Inf, or all NaN
        k = kf.copy()
        k[1, h // G, j, d] = bad                            # a key without weight, or of all rows' NaN, by the query's sign
        check(qf, k, vf, np.s_[1, :, h // G * G:(h // G + 1) * G])
        v = vf.copy()
        v[1, h // G, j, d] = bad                            # that dim of those heads
        check(qf, kf, v, np.s_[1, :, h // G * G:(h // G + 1) * G, d])


def bits(x, t):
    """cast(), with Inf and NaN kept"""
    if t == "f16":
        return cast(x, t)
    u = np.where(np.isfinite(x), mx4.bf16_bits(np.where(np.isfinite(x), x, 0)),
                 np.where(np.isnan(x), 0x7FC0, np.where(x > 0, 0x7F80, 0xFF80))).astype(np.uint16)
    return u, mx4.bf16_value(u)


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("B,H,Hkv,Nq,Nk,D", FORMS)
def test_no_score_above_minus_infinity(hip, t, B, H, Hkv, Nq, Nk, D):
    """A row whose valid keys all score -Inf is zero, like one without valid keys; its neighbours are as they would be."""
    print(f"[gpu] all -inf {t} {Nq} {Nk} {D}", flush=True)
    r = rng(Nq)
    qf, kf, vf = np.abs(randn(r, (B, H, Nq, D))) + 0.25, randn(r, (B, Hkv, Nk, D)), randn(r, (B, Hkv, Nk, D))
    kf[B - 1, :, :, 7] = -np.inf                            # the last sequence's keys
    qf[0, 0, 0] = 0.5
    (q, qv), (k, kv), (v, vv) = bits(qf, t), bits(kf, t), bits(vf, t)
    got = run(hip, t, q, k, v)
    assert (got[B - 1] == 0).all()
    if B > 1:
        want, mag = mx4.cross_attention(qv[:-1], kv[:-1], vv[:-1])
        assert (np.abs(got[:-1] - want) <= tolerance(want, mag, qv[:-1], kv[:-1], vv, t, t, 1 / np.sqrt(D), Nk)).all()
    kf[B - 1, :, Nk // 2] = 0.25                            # one key of a finite score: it alone counts
    k, kv = bits(kf, t)
    got = run(hip, t, q, k, v)
    alone = np.repeat(vv[B - 1, :, Nk // 2], H // Hkv, 0)
    assert np.array_equal(got[B - 1], np.broadcast_to(alone, got[B - 1].shape))
