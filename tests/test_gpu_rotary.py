"""Rotary positions (dl4s_hip_rotary_f32, dl4s_hip_rotary_append_f32, dl4s_hip_rotary_frequencies) against the formula in
64 bits.

Bound of an output: cos and sin are off by at most 2^-23 (the rounding of an angle of at most an eighth of a turn, the
series' rounding), times the amplitude two roundings more, and the two products and their sum round once each:
|y - exact| <= 8 * 2^-24 * amplitude * (|x_a| + |x_b|)."""
import ctypes as C
import math

import numpy as np
import pytest

U = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    from dl4s_amd import lib
    c = lib.Context(0)
    yield c
    c.close()


def _frequencies(rot, base, scaling=0, factor=1.0, low=1.0, high=32.0, original=0):
    if scaling == 2 and rot > 2:
        base = base * factor ** (rot / (rot - 2))
    f = np.array([base ** (-2 * i / rot) for i in range(rot // 2)]) / (2 * math.pi)
    if scaling == 1:
        f = f / factor
    if scaling == 3:
        keep = np.clip((original * f - low) / (high - low), 0, 1)
        f = keep * f + (1 - keep) * f / factor
    return f


def _turned(x, positions, turns, rot, interleaved, amplitude=1.0, inverse=False):
    """x [..., L, d] by positions [..., L]; returns value and bound."""
    x = x.astype(np.float64)
    angle = 2 * np.pi * np.remainder(positions.astype(np.float64)[..., None] * turns, 1.0)
    c, s = np.cos(angle) * amplitude, np.sin(angle) * amplitude * (-1 if inverse else 1)
    y, bound = x.copy(), np.zeros_like(x)
    i = np.arange(rot // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    bound[..., a] = bound[..., b] = 8 * U * abs(amplitude) * (np.abs(x[..., a]) + np.abs(x[..., b]))
    return y, bound


def _within(got, want, what):
    off = np.abs(got.astype(np.float64) - want[0])
    bad = ~(off <= want[1])
    assert not bad.any(), "%s: %d of %d outside, worst %.3g" % (what, bad.sum(), bad.size, np.nanmax(off - want[1]))


def _lay(x, token_major):
    return np.ascontiguousarray(x.transpose(0, 2, 1, 3)) if token_major else x


# ---- the table of frequencies is host arithmetic: checked without a GPU

@pytest.mark.parametrize("rot,kw", [
    (2, {}), (64, {}), (128, dict(scaling=1, factor=4.0)), (64, dict(scaling=2, factor=8.0)), (2, dict(scaling=2, factor=8.0)),
    (128, dict(scaling=3, factor=32.0, low=1.0, high=4.0, original_length=8192)), (0, {})])
def test_frequencies(rot, kw):
    from dl4s_amd import lib
    want = _frequencies(rot, 500000.0, kw.get("scaling", 0), kw.get("factor", 1.0), kw.get("low", 1.0), kw.get("high", 32.0),
                        kw.get("original_length", 0))
    got = lib.rotary_frequencies(rot, 500000.0, **kw)
    assert got.shape == want.shape and np.allclose(got, want, rtol=1e-14, atol=0)


@pytest.mark.parametrize("args,code", [
    ((3, 1e4, 0, 1.0, 1.0, 2.0, 0), -2), ((-2, 1e4, 0, 1.0, 1.0, 2.0, 0), -2), ((4, 0.0, 0, 1.0, 1.0, 2.0, 0), -1),
    ((4, 1e4, 1, 0.0, 1.0, 2.0, 0), -1), ((4, 1e4, 9, 1.0, 1.0, 2.0, 0), -1), ((4, 1e4, 3, 2.0, 2.0, 2.0, 100), -1),
    ((4, 1e4, 3, 2.0, 1.0, 2.0, 0), -1), ((4, float("nan"), 0, 1.0, 1.0, 2.0, 0), -1)])
def test_frequency_refusals(args, code):
    from dl4s_amd import lib
    with pytest.raises(lib.Dl4sHipError) as e:
        lib.rotary_frequencies(*args)
    assert e.value.code == code


# ---- the kernels

@pytest.mark.gpu
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("B,L,H,Hkv,d,rot", [
    (1, 1, 1, 1, 2, 2), (2, 7, 3, 1, 64, 64), (1, 130, 4, 4, 128, 64), (3, 5, 2, 2, 80, 80), (2, 33, 5, 5, 33, 6), (1, 4, 2, 1, 7, 0),
    (2, 3, 8, 2, 256, 256), (1, 9, 2, 1, 96, 20), (2, 6, 0, 3, 64, 32), (2, 6, 3, 0, 64, 64), (1, 65, 33, 3, 20, 12)])
def test_rotary(ctx, B, L, H, Hkv, d, rot, token_major, interleaved, inverse):
    from dl4s_amd import lib
    rng = np.random.default_rng(L * d + H)
    q, k = rng.standard_normal((B, H, L, d)).astype(np.float32), rng.standard_normal((B, Hkv, L, d)).astype(np.float32)
    positions = rng.integers(-50, 200000, (B, L))
    turns = _frequencies(rot, 10000.0)
    flags = interleaved * lib.ROTARY_INTERLEAVED | inverse * lib.ROTARY_INVERSE | token_major * lib.ROTARY_TOKEN_MAJOR
    dq, dk = ctx.to_device(_lay(q, token_major)), ctx.to_device(_lay(k, token_major))
    oq, ok = ctx.empty(dq.shape), ctx.empty(dk.shape)
    dt, dp = ctx.to_device(turns, np.float64), ctx.to_device(positions, np.int32)
    ctx.rotary(dq if H else None, oq if H else None, dk if Hkv else None, ok if Hkv else None, B, L, H, Hkv, d, rot, dt, positions=dp,
               amplitude=1.25, flags=flags)
    for x, o, n in ((q, oq, H), (k, ok, Hkv)):
        if n:
            _within(_lay(o.numpy(), token_major), _turned(x, positions[:, None], turns, rot, interleaved, 1.25, inverse), "turned")
    # in place, the same bits
    ctx.rotary(dq if H else None, dq if H else None, dk if Hkv else None, dk if Hkv else None, B, L, H, Hkv, d, rot, dt, positions=dp,
               amplitude=1.25, flags=flags)
    for x, o, n in ((dq, oq, H), (dk, ok, Hkv)):
        assert not n or np.array_equal(x.numpy(), o.numpy())
    # positions counted from a first one, and back again: the inverse undoes the turn
    ctx.rotary(oq if H else None, oq if H else None, ok if Hkv else None, ok if Hkv else None, B, L, H, Hkv, d, rot, dt, positions=dp,
               flags=flags ^ lib.ROTARY_INVERSE, amplitude=0.8)
    for x, o, n in ((q, oq, H), (k, ok, Hkv)):
        if n:
            got = _lay(o.numpy(), token_major)
            bound = np.full(x.shape, 32 * U * (np.abs(x).max() * 2 + 1))
            _within(got[..., :rot], (x[..., :rot].astype(np.float64), bound[..., :rot]), "there and back")
    for b in (dq, dk, oq, ok, dt, dp):
        b.release()


@pytest.mark.gpu
def test_far_positions_keep_their_precision(ctx):
    """At position 2^30 - 1 the fastest pair has made 1.7e8 turns: 64 bits still hold the angle to 2^-24 of a turn."""
    from dl4s_amd import lib
    L, d = 3, 64
    x = np.random.default_rng(0).standard_normal((1, 1, L, d)).astype(np.float32)
    turns = _frequencies(d, 10000.0)
    dx, out, dt = ctx.to_device(x), ctx.empty(x.shape), ctx.to_device(turns, np.float64)
    first = (1 << 30) - 4
    ctx.rotary(dx, out, None, None, 1, L, 1, 0, d, d, dt, position0=first)
    from fractions import Fraction
    exact = np.array([[float(Fraction(float(t)) * (first + l) % 1) for t in turns] for l in range(L)])
    c, s = np.cos(2 * np.pi * exact), np.sin(2 * np.pi * exact)
    a, b = x[0, 0, :, :32].astype(np.float64), x[0, 0, :, 32:].astype(np.float64)
    bound = (8 * U + 2 * np.pi * 2.0 ** -24) * (np.abs(a) + np.abs(b))
    got = out.numpy()[0, 0]
    _within(got[:, :32], (a * c - b * s, bound), "far")
    _within(got[:, 32:], (a * s + b * c, bound), "far")
    for z in (dx, out, dt):
        z.release()


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("B,L,H,Hkv,d,rot,Tcap", [
    (1, 1, 1, 1, 2, 2, 5), (4, 1, 8, 2, 64, 64, 40), (3, 9, 4, 4, 128, 64, 33), (2, 17, 6, 3, 33, 10, 64), (2, 5, 2, 1, 96, 0, 20),
    (5, 1, 4, 4, 80, 80, 300), (2, 40, 3, 1, 256, 256, 50)])
def test_append(ctx, B, L, H, Hkv, d, rot, Tcap, token_major, interleaved):
    from dl4s_amd import lib
    rng = np.random.default_rng(B * L + d)
    q = rng.standard_normal((B, H, L, d)).astype(np.float32)
    k, v = (rng.standard_normal((B, Hkv, L, d)).astype(np.float32) for _ in range(2))
    kc, vc = (rng.standard_normal((B, Hkv, Tcap, d)).astype(np.float32) for _ in range(2))
    starts = rng.integers(0, Tcap, B)
    starts[0], starts[-1] = Tcap - L, -3 if B > 1 else Tcap - L       # some rows fall outside the cache at either end
    counts = rng.integers(0, L + 1, B)
    counts[0] = L + 5
    turns = _frequencies(rot, 10000.0)
    rows = starts[:, None] + np.arange(L)
    k_turned, k_bound = _turned(k, rows[:, None], turns, rot, interleaved, 0.9)
    flags = interleaved * lib.ROTARY_INTERLEAVED | token_major * lib.ROTARY_TOKEN_MAJOR
    bufs = [ctx.to_device(_lay(x, token_major)) for x in (q, k, v)]
    qo, dt = ctx.empty(bufs[0].shape), ctx.to_device(turns, np.float64)
    dp, dn = ctx.to_device(starts, np.int32), ctx.to_device(counts, np.int32)
    for n in (None, dn):
        dkc, dvc = ctx.to_device(kc), ctx.to_device(vc)
        ctx.rotary_append(*bufs, qo, dkc, dvc, B, L, H, Hkv, Tcap, d, rot, dt, positions=dp, counts=n, amplitude=0.9, flags=flags)
        want_k, bound, want_v = kc.astype(np.float64), np.zeros(kc.shape), vc.copy()
        for b in range(B):
            for l in range(L if n is None else min(L, counts[b])):
                if 0 <= rows[b, l] < Tcap:
                    want_k[b, :, rows[b, l]], bound[b, :, rows[b, l]] = k_turned[b, :, l], k_bound[b, :, l]
                    want_v[b, :, rows[b, l]] = v[b, :, l]
        _within(dkc.numpy(), (want_k, bound), "key cache")
        assert np.array_equal(dvc.numpy(), want_v)
        _within(_lay(qo.numpy(), token_major), _turned(q, rows[:, None], turns, rot, interleaved, 0.9), "queries")
        dkc.release()
        dvc.release()
    for b in bufs + [qo, dt, dp, dn]:
        b.release()


@pytest.mark.gpu
def test_unaligned(ctx):
    rng = np.random.default_rng(2)
    L, d = 11, 64
    x = rng.standard_normal((1, 1, L, d)).astype(np.float32)
    turns = _frequencies(d, 10000.0)
    dx, out, dt = ctx.to_device(np.concatenate([[0], x.ravel()])), ctx.empty((L * d + 1,)), ctx.to_device(turns, np.float64)
    for il in (0, 1):
        ctx.rotary(dx.offset(4), out.offset(4), None, None, 1, L, 1, 0, d, d, dt, flags=il)
        _within(out.numpy()[1:].reshape(x.shape), _turned(x, np.arange(L)[None, None], turns, d, il), "unaligned")
    for z in (dx, out, dt):
        z.release()


@pytest.mark.gpu
@pytest.mark.parametrize("change,code", [(dict(rot=3), -2), (dict(rot=18), -2), (dict(rot=-2), -2), (dict(flags=8), -1), (dict(B=-1), -1),
                                         (dict(null=True), -1), (dict(d=0), -5), (dict(position0=1 << 40), -5)])
def test_refusals(ctx, change, code):
    from dl4s_amd import lib
    a = dict(B=1, L=2, H=1, Hkv=1, d=16, rot=8, flags=0, null=False, position0=0)
    a.update(change)
    x = ctx.empty((256,))
    p = None if a["null"] else x
    with pytest.raises(lib.Dl4sHipError) as e:
        ctx.rotary(p, x, p, x, a["B"], a["L"], a["H"], a["Hkv"], a["d"], a["rot"], x, position0=a["position0"], flags=a["flags"])
    assert e.value.code == code
    with pytest.raises(lib.Dl4sHipError) as e:
        ctx.rotary_append(p, p, p, x, x, x, a["B"], a["L"], a["H"], a["Hkv"], 4, a["d"], a["rot"], x, position0=a["position0"],
                          flags=a["flags"])
    assert e.value.code == code
    with pytest.raises(lib.Dl4sHipError) as e:
        ctx.rotary_append(x, x, x, x, x, x, 1, 1, 1, 1, 4, 16, 8, x, flags=lib.ROTARY_INVERSE)
    assert e.value.code == -1
    x.release()
