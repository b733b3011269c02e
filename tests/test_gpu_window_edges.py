"""Windowed attention at its edges: magnitudes far from one, rows of unlike sizes, what stands in masked places, many visible
first keys, few queries over many keys, offsets past 32 bits, limits.  Bounds: window_reference."""
import ctypes as C

import numpy as np
import pytest

from window_reference import assert_within, attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from dl4s_amd import lib
    c = lib.Context(0)
    yield c
    c.close()


def _inputs(rng, B, H, Hkv, Lq, Lk, d):
    q, g = (rng.standard_normal((B, H, Lq, d)) for _ in range(2))
    k, v = (rng.standard_normal((B, Hkv, Lk, d)) for _ in range(2))
    return [x.astype(np.float32) for x in (q, k, v, g)]


def _forward_backward(ctx, q, k, v, g, rT, window, sinks=0, q_offset=0, lengths=None):
    """{name: array} of out, dq, dk, dv from the device, head-major tensors."""
    B, H, Lq, d = q.shape
    Hkv, Lk = k.shape[1], k.shape[2]
    bufs = [ctx.to_device(x) for x in (q, k, v, g)]
    out, stats, dq, dk, dv = (ctx.to_device(np.full(s, np.nan)) for s in (q.shape, (B, H, Lq, 2), q.shape, k.shape, k.shape))
    ln = None if lengths is None else ctx.to_device(np.asarray(lengths), np.int32)
    args = (B, H, Hkv, Lq, Lk, d, rT, ctx.window_desc(window, sinks, q_offset, ln))
    ctx.sdpa_window_fwd(*bufs[:3], out, stats, *args)
    ctx.sdpa_window_bwd(*bufs[:3], out, stats, bufs[3], dq, dk, dv, *args)
    res = dict(out=out.numpy(), dq=dq.numpy(), dk=dk.numpy(), dv=dv.numpy())
    for b in bufs + [out, stats, dq, dk, dv] + ([ln] if ln is not None else []):
        b.release()
    return res


def _compare(got, want, what):
    for name in got:
        assert_within(got[name], want[name], what + " " + name)


@pytest.mark.parametrize("d", [32, 64, 96, 128, 160])
@pytest.mark.parametrize("sq,sk,sv,sg", [
    (2.0 ** -70, 2.0 ** 70, 1, 1), (2.0 ** 90, 2.0 ** -90, 1, 1), (2.0 ** -60, 2.0 ** -60, 1, 1), (1, 1, 2.0 ** -90, 2.0 ** 60),
    (1, 1, 2.0 ** 90, 2.0 ** -60), (1, 1, 1, 2.0 ** -85), (1, 1, 1, 2.0 ** 100), (2.0 ** -20, 2.0 ** 20, 2.0 ** -85, 1), (0, 1, 1, 1),
    (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1, 0)])
def test_magnitudes(ctx, sq, sk, sv, sg, d):
    """Tensors of any size in fp32's range, and tensors of zeros."""
    rng = np.random.default_rng(d)
    q, k, v, g = (x * np.float32(s) for x, s in zip(_inputs(rng, 1, 4, 2, 150, 150, d), (sq, sk, sv, sg)))
    rT = float(np.float32(1 / np.sqrt(d)))
    got = _forward_backward(ctx, q, k, v, g, rT, 40, 5)
    _compare(got, attention(q, k, v, rT, 40, 5, dout=g), "scales %g %g %g %g" % (sq, sk, sv, sg))


@pytest.mark.parametrize("rT", [0.0, -0.3, 2.0 ** -100, 2.0 ** -40])
def test_temperatures(ctx, rT):
    rng = np.random.default_rng(1)
    q, k, v, g = _inputs(rng, 1, 2, 1, 90, 90, 64)
    q *= np.float32(1 if abs(rT) > 1e-3 or rT == 0 else 0.125 / rT)
    _compare(_forward_backward(ctx, q, k, v, g, rT, 30, 2), attention(q, k, v, rT, 30, 2, dout=g), "temperature %g" % rT)


@pytest.mark.parametrize("d", [64, 96, 128])
def test_rows_of_unlike_sizes(ctx, d):
    """Every row has a power of two of its own, between 2^-4 and 2^4; a value's error is then at most a step of fp32's."""
    rng = np.random.default_rng(d)
    q, k, v, g = (x * np.exp2(rng.integers(-4, 5, x.shape[:3] + (1,))).astype(np.float32) for x in _inputs(rng, 2, 4, 2, 200, 200, d))
    rT = 1 / 32.0
    _compare(_forward_backward(ctx, q, k, v, g, rT, 70, 3), attention(q, k, v, rT, 70, 3, dout=g), "unlike rows")


@pytest.mark.parametrize("d", [64, 100, 160])
@pytest.mark.parametrize("Lq", [40, 100])
def test_keys_that_no_query_sees(ctx, Lq, d):
    """Rows of a cache before the first window (behind the visible first keys), and behind the last query, may hold anything."""
    rng = np.random.default_rng(7)
    B, H, Hkv, Lk, window, sinks, offset = 2, 2, 1, 400, 33, 4, 200
    q, k, v, g = _inputs(rng, B, H, Hkv, Lq, Lk, d)
    hidden = np.r_[sinks:offset - window + 1, offset + Lq:Lk]
    want = attention(q, k, v, 0.1, window, sinks, offset, dout=g)
    k[:, :, hidden], v[:, :, hidden] = np.nan, np.inf
    _compare(_forward_backward(ctx, q, k, v, g, 0.1, window, sinks, offset), want, "hidden keys")


@pytest.mark.parametrize("d", [64, 96, 160])
def test_rows_that_see_no_key(ctx, d):
    """A window behind the last valid key: whatever the query and its upstream gradient hold, nothing comes of it."""
    rng = np.random.default_rng(9)
    B, H, Hkv, L, window, lengths = 2, 2, 1, 160, 20, [50, 0]
    q, k, v, g = _inputs(rng, B, H, Hkv, L, L, d)
    want = attention(q, k, v, 0.1, window, 0, 0, lengths, g)
    q[0, :, 69:], g[0, :, 69:] = np.nan, np.inf
    q[1], g[1] = np.inf, np.nan
    k[0, :, 50:], v[0, :, 50:], k[1], v[1] = np.nan, np.nan, np.inf, np.nan
    got = _forward_backward(ctx, q, k, v, g, 0.1, window, 0, 0, lengths)
    _compare(got, want, "empty rows")
    assert not got["out"][0, :, 69:].any() and not got["dq"][0, :, 69:].any() and not got["dk"][1].any()


def test_a_value_that_is_not_a_number_reaches_the_rows_that_see_it(ctx):
    rng = np.random.default_rng(10)
    q, k, v, g = _inputs(rng, 1, 1, 1, 200, 200, 64)
    q[0, 0, 77] = np.nan
    got = _forward_backward(ctx, q, k, v, g, 0.125, 30)
    assert np.isnan(got["out"][0, 0, 77]).all() and np.isfinite(np.delete(got["out"][0, 0], 77, 0)).all()
    assert np.isnan(got["dq"][0, 0, 77]).all() and np.isnan(got["dv"][0, 0, 48:78]).all()
    assert np.isfinite(got["dv"][0, 0, :48]).all() and np.isfinite(got["dv"][0, 0, 78:]).all()


@pytest.mark.parametrize("d", [40, 64, 96, 128])
@pytest.mark.parametrize("B,H,Hkv,Lq,Lk,window,sinks", [
    (1, 1, 1, 1000, 1000, 10, 300), (1, 4, 1, 700, 700, 50, 700), (1, 2, 2, 520, 520, 1, 129), (1, 8, 2, 1100, 1100, 300, 4),
    (1, 1, 1, 2500, 2500, 2500, 0)])
def test_many_first_keys_and_long_windows(ctx, B, H, Hkv, Lq, Lk, window, sinks, d):
    """Key blocks whose queries are dealt to several workgroups."""
    rng = np.random.default_rng(Lq + d)
    q, k, v, g = _inputs(rng, B, H, Hkv, Lq, Lk, d)
    rT = float(np.float32(1 / np.sqrt(d)))
    _compare(_forward_backward(ctx, q, k, v, g, rT, window, sinks, Lk - Lq), attention(q, k, v, rT, window, sinks, Lk - Lq, dout=g), "first keys")


@pytest.mark.parametrize("d", [64, 80, 128, 256])
@pytest.mark.parametrize("B,H,Hkv,Lq,Lk,window,sinks,lengths", [
    (1, 2, 1, 3, 3000, 5000, 0, None), (2, 4, 2, 16, 2000, 900, 5, [2000, 1500]), (1, 1, 1, 32, 5000, 4000, 40, [4990]),
    (1, 3, 3, 40, 4000, 4000, 0, None), (1, 8, 1, 64, 2500, 2500, 3, None), (1, 16, 2, 2, 1200, 700, 0, [300])])
def test_few_queries_over_many_keys(ctx, B, H, Hkv, Lq, Lk, window, sinks, lengths, d):
    rng = np.random.default_rng(Lk + Lq + d)
    q, k, v, g = _inputs(rng, B, H, Hkv, Lq, Lk, d)
    rT = float(np.float32(1 / np.sqrt(d)))
    want = attention(q, k, v, rT, window, sinks, Lk - Lq, lengths, g)
    _compare(_forward_backward(ctx, q, k, v, g, rT, window, sinks, Lk - Lq, lengths), want, "few queries")


@pytest.mark.parametrize("d", [64, 256])
def test_groups_of_different_sizes_in_turn(ctx, d):
    """The wider a group, the more shared memory a decoding step takes: any order of them works."""
    rng = np.random.default_rng(12)
    for H in (8, 16, 9, 40):
        q, k, v = rng.standard_normal((1, H, 1, d)), rng.standard_normal((1, 1, 50, d)), rng.standard_normal((1, 1, 50, d))
        q, k, v = (x.astype(np.float32) for x in (q, k, v))
        bufs, out = [ctx.to_device(x) for x in (q, k, v)], ctx.empty(q.shape)
        ctx.sdpa_window_decode(*bufs, out, 1, H, 1, 50, 50, d, 0.1, 20)
        assert_within(out.numpy(), attention(q, k, v, 0.1, 20, 0, 49)["out"], "group of %d" % H)
        for b in bufs + [out]:
            b.release()


def test_keys_and_values_may_be_one_tensor(ctx):
    rng = np.random.default_rng(13)
    q, k, _, g = _inputs(rng, 1, 2, 2, 120, 120, 64)
    bufs = [ctx.to_device(x) for x in (q, k, g)]
    out, stats, dq, dk, dv = (ctx.empty(s) for s in (q.shape, (1, 2, 120, 2), q.shape, k.shape, k.shape))
    args = (1, 2, 2, 120, 120, 64, 0.125, ctx.window_desc(50))
    ctx.sdpa_window_fwd(bufs[0], bufs[1], bufs[1], out, stats, *args)
    ctx.sdpa_window_bwd(bufs[0], bufs[1], bufs[1], out, stats, bufs[2], dq, dk, dv, *args)
    _compare(dict(out=out.numpy(), dq=dq.numpy(), dk=dk.numpy(), dv=dv.numpy()), attention(q, k, k, 0.125, 50, dout=g), "one tensor")
    for b in bufs + [out, stats, dq, dk, dv]:
        b.release()


def _copy(ctx, dst, src, nbytes):
    from dl4s_amd import lib
    lib._check(ctx.lib.dl4s_hip_assign_d2d(ctx.handle, C.c_void_p(dst), C.c_void_p(src), C.c_size_t(nbytes)))


def test_decoding_past_32_bit_offsets(ctx):
    """A cache of more than 2^32 elements; its evicted rows hold NaN."""
    B, T, d, window, sinks = 2, (1 << 23) + 77, 256, 300, 5
    rng = np.random.default_rng(14)
    q = rng.standard_normal((B, 1, 1, d)).astype(np.float32)
    near = rng.standard_normal((B, sinks + window, d)).astype(np.float32)
    cache, out, dq = ctx.empty((B, 1, T, d)), ctx.empty(q.shape), ctx.to_device(q)
    for b in range(B):
        ctx.fill(float("nan"), cache.offset(4 * b * T * d), T * d)
        rows = ctx.to_device(near[b])
        _copy(ctx, cache.offset(4 * b * T * d), rows.ptr, 4 * sinks * d)
        _copy(ctx, cache.offset(4 * ((b + 1) * T - window) * d), rows.offset(4 * sinks * d), 4 * window * d)
        rows.release()
    ctx.sdpa_window_decode(dq, cache, cache, out, B, 1, 1, T, T, d, 0.06, window, sinks)
    k = near[:, None]
    assert_within(out.numpy(), attention(q, k, k, 0.06, sinks + window, 0, sinks + window - 1)["out"], "far cache")
    for x in (cache, out, dq):
        x.release()
    ctx.pool_trim(0)


def test_training_past_32_bit_offsets(ctx):
    """Keys and their gradients more than 2^31 elements behind the first one."""
    Lq, Lk, d, window, sinks = 70, (1 << 24) + 200, 128, 90, 2
    rng = np.random.default_rng(15)
    q, g = (rng.standard_normal((1, 1, Lq, d)).astype(np.float32) for _ in range(2))
    seen = sinks + window - 1 + Lq
    near = rng.standard_normal((seen, d)).astype(np.float32)
    keys, rows = ctx.empty((Lk, d)), ctx.to_device(near)
    ctx.fill(float("nan"), keys, Lk * d)
    tail = 4 * (Lk - (seen - sinks)) * d
    _copy(ctx, keys.ptr, rows.ptr, 4 * sinks * d)
    _copy(ctx, keys.offset(tail), rows.offset(4 * sinks * d), 4 * (seen - sinks) * d)
    bufs = [ctx.to_device(q), ctx.to_device(g)]
    out, stats, dq, dk, dv = (ctx.empty(s) for s in (q.shape, (1, 1, Lq, 2), q.shape, (Lk, d), (Lk, d)))
    args = (1, 1, 1, Lq, Lk, d, 0.09, ctx.window_desc(window, sinks, Lk - Lq))
    ctx.sdpa_window_fwd(bufs[0], keys, keys, out, stats, *args)
    ctx.sdpa_window_bwd(bufs[0], keys, keys, out, stats, bufs[1], dq, dk, dv, *args)
    # the same without the rows between: a key's distance to the queries stays what it was
    want = attention(q, near[None, None], near[None, None], 0.09, window, sinks, seen - Lq, None, g)
    got = dict(out=out.numpy(), dq=dq.numpy())
    for name, x in (("dk", dk), ("dv", dv)):
        _copy(ctx, rows.ptr, x.ptr, 4 * sinks * d)
        _copy(ctx, rows.offset(4 * sinks * d), x.offset(tail), 4 * (seen - sinks) * d)
        got[name] = rows.numpy()[None, None]
        _copy(ctx, rows.ptr, x.offset(tail - 4 * seen * d), 4 * seen * d)
        assert not rows.numpy().any()                        # keys that nothing sees
    _compare(got, want, "far keys")
    for x in bufs + [keys, rows, out, stats, dq, dk, dv]:
        x.release()
    ctx.pool_trim(0)


@pytest.mark.parametrize("change", [
    dict(H=1 << 15, Hkv=1 << 15, d=256), dict(q_offset=(1 << 30) - 256), dict(Lq=1 << 30), dict(Lk=(1 << 30) - 100),
    dict(B=1 << 24, Lq=20, Lk=1), dict(H=4, Lq=1 << 29), dict(H=4, Lq=1 << 29, d=200), dict(B=1 << 29, H=4, Hkv=4)])
def test_limits_are_refused(ctx, change):
    """Extents that the kernels' 32-bit positions and offsets, or one launch, do not hold."""
    from dl4s_amd import lib
    a = dict(B=1, H=1, Hkv=1, Lq=40, Lk=40, d=16, q_offset=0)
    a.update(change)
    x = ctx.empty((64,))
    args = (a["B"], a["H"], a["Hkv"], a["Lq"], a["Lk"], a["d"], 1.0, ctx.window_desc(4, 0, a["q_offset"]))
    for call in (lambda: ctx.sdpa_window_fwd(x, x, x, x, None, *args), lambda: ctx.sdpa_window_bwd(x, x, x, x, x, x, x, x, x, *args)):
        with pytest.raises(lib.Dl4sHipError) as e:
            call()
        assert e.value.code == -5
    x.release()


@pytest.mark.parametrize("B,H,Hkv,d", [(70000, 1, 1, 5), (1, 40000, 1, 8), (66000, 1, 1, 140)])
def test_very_many_heads(ctx, B, H, Hkv, d):
    """More (batch, key head) pairs than a grid's second axis has, a group of thousands: decoding and one row of a prompt."""
    rng = np.random.default_rng(16)
    q, k, v, _ = _inputs(rng, B, H, Hkv, 1, 3, d)
    bufs, out = [ctx.to_device(x) for x in (q, k, v)], ctx.empty(q.shape)
    group = q.reshape(B, Hkv, H // Hkv, d).astype(np.float64)
    s = (group @ k[:, :, 1:].astype(np.float64).transpose(0, 1, 3, 2)) * 0.2
    w = np.exp(s - s.max(-1, keepdims=True))
    w /= w.sum(-1, keepdims=True)
    want = (w @ v[:, :, 1:]).reshape(q.shape)
    # worst case of two keys: the scores' errors, their weights', the sum's (window_reference)
    size = (np.abs(group) @ np.abs(k[:, :, 1:]).transpose(0, 1, 3, 2)).max(-1, keepdims=True) * 0.2
    bound = 2.0 ** -24 * ((2 * (d + 24) * (1 + size) + 40) * np.abs(v).max((2, 3))[:, :, None, None]).reshape(B, H, 1, 1)
    for call in (lambda: ctx.sdpa_window_decode(*bufs, out, B, H, Hkv, 3, 3, d, 0.2, 2),
                 lambda: ctx.sdpa_window_fwd(*bufs, out, None, B, H, Hkv, 1, 3, d, 0.2, ctx.window_desc(2, 0, 2))):
        ctx.fill(float("nan"), out, B * H * d)
        call()
        assert (np.abs(out.numpy() - want) <= bound).all()
    for x in bufs + [out]:
        x.release()


def test_limits_of_one_launch(ctx):
    from dl4s_amd import lib
    x = ctx.empty((64,))
    with pytest.raises(lib.Dl4sHipError) as e:            # 2^23 workgroups of 16 rows
        ctx.sdpa_window_fwd(x, x, x, x, None, 1, 1, 1, 1 << 27, 4, 140, 1.0, ctx.window_desc(4))
    assert e.value.code == -5
    x.release()


@pytest.mark.parametrize("d", [32, 60, 64, 96, 97, 128])
@pytest.mark.parametrize("B,H,Hkv,Lq,Lk,window,sinks,lengths", [
    (3, 6, 3, 900, 900, 300, 0, [900, 333, 1]), (1, 16, 4, 700, 700, 700, 7, None), (2, 8, 8, 513, 700, 250, 65, [700, 260]),
    (1, 9, 9, 500, 500, 1000, 0, [0]), (1, 12, 4, 450, 450, 193, 0, None), (8, 8, 8, 520, 520, 220, 3, None)])
def test_small_and_large_launches(ctx, B, H, Hkv, Lq, Lk, window, sinks, lengths, d):
    """Launches of fewer workgroups than compute units, where eight wavefronts share a workgroup's rows, and of more."""
    rng = np.random.default_rng(Lq + d)
    q, k, v, g = _inputs(rng, B, H, Hkv, Lq, Lk, d)
    q[:, :, ::7] *= 8                                      # some rows with one large score, others without
    rT = float(np.float32(1 / np.sqrt(d)))
    want = attention(q, k, v, rT, window, sinks, Lk - Lq, lengths, g)
    _compare(_forward_backward(ctx, q, k, v, g, rT, window, sinks, Lk - Lq, lengths), want, "launches")
