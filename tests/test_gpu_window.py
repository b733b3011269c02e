"""Attention with a sliding window and visible first keys (dl4s_hip_sdpa_window_*) against its formula in 64 bits, inside
bounds that follow from fp32 arithmetic (window_reference)."""
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


def _put(ctx, x, token_major):
    return ctx.to_device(np.ascontiguousarray(x.transpose(0, 2, 1, 3)) if token_major else x)


def _got(buf, token_major):
    x = buf.numpy()
    return x.transpose(0, 2, 1, 3) if token_major else x


def _run(ctx, B, H, Hkv, Lq, Lk, d, window, sinks=0, q_offset=None, lengths=None, token_major=False, train=False, seed=0, scale=1.0):
    from dl4s_amd import lib
    rng = np.random.default_rng(seed)
    q, dout = ((rng.standard_normal((B, H, Lq, d)) * scale).astype(np.float32) for _ in range(2))
    k, v = ((rng.standard_normal((B, Hkv, Lk, d)) * scale).astype(np.float32) for _ in range(2))
    q_offset = Lk - Lq if q_offset is None else q_offset
    rT = float(np.float32(1 / np.sqrt(d)))
    if lengths is not None:
        for b, n in enumerate(lengths):        # whatever stands behind the last valid key stays out
            k[b, :, max(0, n):] = np.nan
            v[b, :, max(0, n):] = np.inf
    want = attention(q, k, v, rT, window, sinks, q_offset, lengths, dout if train else None)
    put = lambda x: _put(ctx, x, token_major)
    dq_, dk_, dv_, do_ = put(q), put(k), put(v), put(dout)
    shape_q, shape_k = dq_.shape, dk_.shape
    out, stats = ctx.empty(shape_q), ctx.empty((B, H, max(Lq, 1), 2))
    ctx.fill(float("nan"), out, int(np.prod(shape_q)))
    ln = None if lengths is None else ctx.to_device(np.asarray(lengths), np.int32)
    desc = ctx.window_desc(window, sinks, q_offset, ln)
    flags = lib.SDPA_TOKEN_MAJOR if token_major else 0
    args = (B, H, Hkv, Lq, Lk, d, rT, desc, flags)
    ctx.sdpa_window_fwd(dq_, dk_, dv_, out, stats if train else None, *args)
    what = "B%d H%d/%d Lq%d Lk%d d%d w%d s%d off%d" % (B, H, Hkv, Lq, Lk, d, window, sinks, q_offset)
    assert_within(_got(out, token_major), want["out"], what + " out")
    bufs = [dq_, dk_, dv_, do_, out, stats]
    if train:
        gq, gk, gv = ctx.empty(shape_q), ctx.empty(shape_k), ctx.empty(shape_k)
        for g, n in ((gq, shape_q), (gk, shape_k), (gv, shape_k)):
            ctx.fill(float("nan"), g, int(np.prod(n)))
        ctx.sdpa_window_bwd(dq_, dk_, dv_, out, stats, do_, gq, gk, gv, *args)
        first = [g.numpy() for g in (gq, gk, gv)]
        for name, g in (("dq", gq), ("dk", gk), ("dv", gv)):
            assert_within(_got(g, token_major), want[name], what + " " + name)
        ctx.sdpa_window_bwd(dq_, dk_, dv_, out, stats, do_, gq, gk, gv, *args)
        for a, g in zip(first, (gq, gk, gv)):
            assert np.array_equal(a, g.numpy()), what + ": another run, other bits"
        bufs += [gq, gk, gv]
    for x in bufs + ([ln] if ln is not None else []):
        x.release()


HEAD_DIMS = [1, 3, 16, 30, 32, 33, 40, 64, 66, 80, 96, 100, 127, 128, 129, 200, 256]


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("d", HEAD_DIMS)
def test_head_dims(ctx, d, train):
    _run(ctx, 2, 4, 2, 70, 70, d, 20, 3, train=train, seed=d)


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("Lq,Lk,window,sinks,q_offset", [
    (1, 1, 1, 0, 0), (1, 1, 7, 2, 0), (2, 2, 1, 0, 0), (33, 33, 1, 0, 0), (33, 33, 1, 1, 0), (31, 31, 1000, 0, 0), (64, 64, 32, 0, 0),
    (128, 128, 32, 4, 0), (129, 129, 33, 5, 0), (257, 257, 64, 64, 0), (300, 300, 17, 40, 0), (300, 300, 2, 299, 0),
    (1, 300, 50, 4, 299), (37, 300, 50, 4, 263), (37, 300, 50, 4, 100), (5, 300, 1, 0, 0), (300, 40, 16, 0, 0), (300, 40, 16, 3, 0),
    (100, 40, 8, 0, 60), (17, 513, 512, 1, 496), (520, 520, 500, 0, 0), (96, 200, 1 << 40, 0, 104), (65, 65, 64, 1 << 40, 0)])
def test_windows(ctx, Lq, Lk, window, sinks, q_offset, train):
    _run(ctx, 1, 2, 1, Lq, Lk, 64, window, sinks, q_offset, train=train, seed=Lq + Lk)


@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (3, 1), (6, 2), (8, 8), (5, 5)])
def test_heads_and_layouts(ctx, H, Hkv, token_major):
    _run(ctx, 3, H, Hkv, 90, 90, 32, 25, 2, token_major=token_major, train=True, seed=H)
    _run(ctx, 2, H, Hkv, 40, 150, 128, 70, 9, token_major=token_major, train=True, seed=H + 1)


@pytest.mark.parametrize("d", [40, 64, 128])
@pytest.mark.parametrize("lengths", [[150, 149, 100, 33], [32, 1, 0, 150], [0, 0, 0, 0], [-5, 700, 64, 65]])
def test_key_lengths(ctx, lengths, d):
    """Windows that lie behind the last valid key leave rows empty: their output is zero, and so is what flows back."""
    _run(ctx, 4, 2, 1, 150, 150, d, 30, 0, lengths=lengths, train=True, seed=1)
    _run(ctx, 4, 2, 2, 150, 150, d, 30, 5, lengths=lengths, train=True, seed=2, token_major=True)


def test_large_scores(ctx):
    """Scores of some hundreds: one key takes nearly all the weight."""
    _run(ctx, 1, 2, 2, 130, 130, 64, 40, 4, train=True, seed=3, scale=4.0)


def test_unaligned_operands(ctx):
    """Pointers four bytes off the 16-byte grid."""
    from dl4s_amd import lib
    rng = np.random.default_rng(8)
    B, H, L, d, window = 1, 2, 80, 64, 30
    host = [rng.standard_normal((B, H, L, d)).astype(np.float32) for _ in range(4)]
    n = B * H * L * d
    bufs = [ctx.to_device(np.concatenate([np.zeros(1, np.float32), x.ravel()])) for x in host]
    outs = [ctx.empty((n + 1,)) for _ in range(4)]
    stats = ctx.empty((B, H, L, 2))
    want = attention(host[0], host[1], host[2], 0.125, window, dout=host[3])
    q, k, v, g = (b.offset(4) for b in bufs)
    o, dq, dk, dv = (b.offset(4) for b in outs)
    args = (B, H, H, L, L, d, 0.125, ctx.window_desc(window))
    ctx.sdpa_window_fwd(q, k, v, o, stats, *args)
    ctx.sdpa_window_bwd(q, k, v, o, stats, g, dq, dk, dv, *args)
    for name, b in zip(("out", "dq", "dk", "dv"), outs):
        assert_within(b.numpy()[1:].reshape(B, H, L, d), want[name], "unaligned " + name)
    for b in bufs + outs + [stats]:
        b.release()


@pytest.mark.parametrize("d", [1, 5, 32, 64, 72, 80, 96, 128, 130, 256])
@pytest.mark.parametrize("B,H,Hkv,T,window,sinks,lengths", [
    (1, 1, 1, 1, 1, 0, None), (2, 4, 2, 40, 1, 0, None), (2, 8, 1, 300, 64, 4, [300, 17]), (3, 6, 2, 700, 5000, 0, [700, 0, 1]),
    (4, 3, 3, 513, 100, 33, [513, 512, 101, 99]), (1, 8, 8, 1500, 1400, 2, [1500])])
def test_decode(ctx, B, H, Hkv, T, window, sinks, lengths, d):
    rng = np.random.default_rng(T + d)
    Tcap = T + 3
    q = rng.standard_normal((B, H, 1, d)).astype(np.float32)
    k, v = (rng.standard_normal((B, Hkv, Tcap, d)).astype(np.float32) for _ in range(2))
    rT = float(np.float32(1 / np.sqrt(d)))
    valid = [T] * B if lengths is None else lengths
    want, bound = np.zeros((B, H, 1, d)), np.zeros((B, H, 1, d))
    for b, n in enumerate(valid):
        k[b, :, n:], v[b, :, n:] = np.nan, np.inf
        if n > 0:
            x = slice(b, b + 1)
            want[b], bound[b] = (y[0] for y in attention(q[x], k[x, :, :n], v[x, :, :n], rT, window, sinks, n - 1)["out"])
    dq, dk, dv, out = ctx.to_device(q), ctx.to_device(k), ctx.to_device(v), ctx.empty(q.shape)
    ctx.fill(float("nan"), out, out.nbytes // 4)
    ln = None if lengths is None else ctx.to_device(np.asarray(lengths), np.int32)
    ctx.sdpa_window_decode(dq, dk, dv, out, B, H, Hkv, T, Tcap, d, rT, window, sinks, ln)
    assert_within(out.numpy(), (want, bound), "decode T%d d%d w%d s%d" % (T, d, window, sinks))
    for x in [dq, dk, dv, out] + ([ln] if ln is not None else []):
        x.release()


def test_agrees_with_causal_attention(ctx):
    """A window that reaches back to the first key is the causal mask of dl4s_hip_sdpa_fwd_f32."""
    from dl4s_amd import lib
    rng = np.random.default_rng(4)
    B, H, L, d = 2, 3, 200, 64
    q, k, v = (rng.standard_normal((B, H, L, d)).astype(np.float32) for _ in range(3))
    bufs = [ctx.to_device(x) for x in (q, k, v)]
    a, b = ctx.empty(q.shape), ctx.empty(q.shape)
    ctx.sdpa_fwd(*bufs, a, B, H, L, L, d, d, 0.125, ctx.mask_desc(lib.MASK_CAUSAL))
    ctx.sdpa_window_fwd(*bufs, b, None, B, H, H, L, L, d, 0.125, ctx.window_desc(L))
    want = attention(q, k, v, 0.125, L)["out"]
    assert_within(b.numpy(), want, "window of the whole length")
    assert_within(a.numpy(), want, "causal")
    for x in bufs + [a, b]:
        x.release()


def test_gradients_by_differences(ctx):
    """A directional derivative of sum(out * dout) by central differences: with step h = 2^-6 along unit-sized directions the
    difference quotient is off by O(h^2) of the third derivative (a few tenths at these sizes) plus the outputs' own error
    over h, together below 1 % of a derivative that is a sum of thousands of terms."""
    from dl4s_amd import lib
    rng = np.random.default_rng(11)
    B, H, Hkv, L, d, window, sinks = 1, 4, 2, 75, 48, 20, 3
    q, g, uq = (rng.standard_normal((B, H, L, d)) for _ in range(3))
    k, v, uk, uv = (rng.standard_normal((B, Hkv, L, d)) for _ in range(4))
    f32 = lambda x: ctx.to_device(x.astype(np.float32))
    rT, desc = 1 / np.sqrt(d), ctx.window_desc(window, sinks)
    out, stats = ctx.empty(q.shape), ctx.empty((B, H, L, 2))

    def value(t):
        bufs = [f32(q + t * uq), f32(k + t * uk), f32(v + t * uv)]
        ctx.sdpa_window_fwd(*bufs, out, stats, B, H, Hkv, L, L, d, rT, desc)
        r = float((out.numpy().astype(np.float64) * g).sum())
        for b in bufs:
            b.release()
        return r

    h = 2.0 ** -6
    slope = (value(h) - value(-h)) / (2 * h)
    slope2 = (value(2 * h) - value(-2 * h)) / (4 * h)
    slope = slope + (slope - slope2) / 3                       # the h^2 term taken off
    value(0.0)
    bufs = [f32(q), f32(k), f32(v), f32(g)]
    grads = [ctx.empty(q.shape), ctx.empty(k.shape), ctx.empty(k.shape)]
    ctx.sdpa_window_fwd(*bufs[:3], out, stats, B, H, Hkv, L, L, d, rT, desc)
    ctx.sdpa_window_bwd(*bufs[:3], out, stats, bufs[3], *grads, B, H, Hkv, L, L, d, rT, desc)
    parts = [float((x.numpy().astype(np.float64) * u).sum()) for x, u in zip(grads, (uq, uk, uv))]
    assert abs(slope - sum(parts)) <= 0.01 * sum(abs(p) for p in parts), (slope, parts)
    for b in bufs + grads + [out, stats]:
        b.release()


def test_nothing_to_do(ctx):
    x = ctx.empty((4,))
    desc = ctx.window_desc(3)
    ctx.sdpa_window_fwd(x, x, x, x, None, 0, 2, 2, 4, 4, 8, 1.0, desc)
    ctx.sdpa_window_fwd(x, x, x, x, None, 1, 2, 2, 0, 4, 8, 1.0, desc)
    ctx.sdpa_window_decode(x, x, x, x, 0, 2, 2, 1, 1, 8, 1.0, 3)
    out = ctx.to_device(np.full((1, 1, 3, 2), np.nan))
    q = ctx.to_device(np.ones((1, 1, 3, 2)))
    ctx.sdpa_window_fwd(q, x, x, out, None, 1, 1, 1, 3, 0, 2, 1.0, desc)      # queries without any key
    assert np.array_equal(out.numpy(), np.zeros((1, 1, 3, 2)))
    for b in (x, out, q):
        b.release()


@pytest.mark.parametrize("change,code", [
    (dict(window=0), -1), (dict(sinks=-1), -1), (dict(q_offset=-1), -1), (dict(flags=1), -1), (dict(flags=4), -1), (dict(Hkv=3), -2),
    (dict(Hkv=0), -2), (dict(d=0), -5), (dict(d=257), -5), (dict(B=-1), -1), (dict(Lk=1 << 31), -5), (dict(null=True), -1)])
def test_refusals(ctx, change, code):
    from dl4s_amd import lib
    a = dict(B=1, H=4, Hkv=2, Lq=8, Lk=8, d=16, window=4, sinks=0, q_offset=0, flags=0, null=False)
    a.update(change)
    x = ctx.empty((1 * 4 * 8 * 16 * 2,))
    p = None if a["null"] else x
    desc = ctx.window_desc(a["window"], a["sinks"], a["q_offset"])
    shape = (a["B"], a["H"], a["Hkv"], a["Lq"], a["Lk"], a["d"], 1.0, desc, a["flags"])
    ptr = 0 if p is None else p.ptr
    for call in (lambda: ctx.sdpa_window_fwd(ptr, ptr, ptr, x, None, *shape),
                 lambda: ctx.sdpa_window_bwd(ptr, ptr, ptr, x, x, x, x, x, x, *shape)):
        with pytest.raises(lib.Dl4sHipError) as e:
            call()
        assert e.value.code == code
    x.release()


@pytest.mark.parametrize("change,code", [(dict(T=9), -2), (dict(T=0), -2), (dict(window=0), -1), (dict(Hkv=3), -2), (dict(d=300), -5)])
def test_decode_refusals(ctx, change, code):
    from dl4s_amd import lib
    a = dict(B=1, H=4, Hkv=2, T=8, Tcap=8, d=16, window=4)
    a.update(change)
    x = ctx.empty((1024,))
    with pytest.raises(lib.Dl4sHipError) as e:
        ctx.sdpa_window_decode(x, x, x, x, a["B"], a["H"], a["Hkv"], a["T"], a["Tcap"], a["d"], 1.0, a["window"])
    assert e.value.code == code
    x.release()


def test_a_missing_descriptor_is_refused(ctx):
    import ctypes as C
    null = C.c_void_p(None)
    i = C.c_int64
    rc = ctx.lib.dl4s_hip_sdpa_window_fwd_f32(ctx.handle, null, null, null, null, null, i(1), i(1), i(1), i(1), i(1), i(8), C.c_float(1),
                                              None, C.c_uint32(0))
    assert rc == -1 and b"descriptor" in ctx.lib.dl4s_hip_last_error()
