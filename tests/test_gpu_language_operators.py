"""The operators of a language model together, as a model has them: rotary positions, windowed attention, the output layer, the
log probabilities and all their gradients; a prompt and the steps after it over one cache; the same calls recorded and
replayed; two contexts at once."""
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


def _f32(rng, *shape):
    return rng.standard_normal(shape).astype(np.float32)


class Model:
    """q, k, v [B,H|Hkv,L,d] -> rotary -> windowed attention -> logits over V tokens -> mean log probability + entropy."""
    B, H, Hkv, L, d, V, window, sinks = 2, 4, 2, 50, 32, 300, 13, 2

    def __init__(self, ctx):
        from dl4s_amd import lib
        self.ctx, self.rows = ctx, self.B * self.L
        self.D = self.H * self.d
        rng = np.random.default_rng(21)
        self.turns = ctx.to_device(lib.rotary_frequencies(self.d), np.float64)
        self.targets = ctx.to_device(rng.integers(0, self.V, self.rows), np.int32)
        self.w = ctx.to_device(_f32(rng, self.D, self.V) * 0.1)
        self.dlp = ctx.to_device(_f32(rng, self.rows))
        self.dent = ctx.to_device(_f32(rng, self.rows))
        e = lambda *s: ctx.empty(s)
        self.qr, self.kr = e(self.B, self.L, self.H, self.d), e(self.B, self.L, self.Hkv, self.d)
        self.out, self.stats = e(self.B, self.L, self.H, self.d), e(self.B, self.H, self.L, 2)
        self.logits, self.lp, self.ent, self.lstats = e(self.rows, self.V), e(self.rows), e(self.rows), e(self.rows, 3)
        self.dlogits, self.dout = e(self.rows, self.V), e(self.B, self.L, self.H, self.d)
        self.dq, self.dk, self.dv = e(self.B, self.L, self.H, self.d), e(self.B, self.L, self.Hkv, self.d), e(self.B, self.L, self.Hkv, self.d)
        self.desc = ctx.window_desc(self.window, self.sinks)
        self.flags = lib.SDPA_TOKEN_MAJOR
        self.rflags, self.rinverse = lib.ROTARY_TOKEN_MAJOR, lib.ROTARY_TOKEN_MAJOR | lib.ROTARY_INVERSE
        self.shape = (self.B, self.H, self.Hkv, self.L, self.L, self.d, float(np.float32(self.d ** -0.5)), self.desc, self.flags)

    def forward(self, q, k, v):
        c = self.ctx
        c.rotary(q, self.qr, k, self.kr, self.B, self.L, self.H, self.Hkv, self.d, self.d, self.turns, flags=self.rflags)
        c.sdpa_window_fwd(self.qr, self.kr, v, self.out, self.stats, *self.shape)
        c.gemm(self.out, (self.rows, self.D), self.w, (self.D, self.V), self.logits)
        c.token_logprobs(self.logits, self.rows, self.V, self.V, self.targets, self.lp, entropy=self.ent, stats=self.lstats)

    def backward(self, q, k, v):
        c = self.ctx
        c.token_logprobs_bwd(self.logits, self.rows, self.V, self.V, self.targets, self.lstats, self.dlogits, dlogprobs=self.dlp, dentropy=self.dent)
        c.gemm(self.dlogits, (self.rows, self.V), self.w, (self.D, self.V), self.dout, tb=True)
        c.sdpa_window_bwd(self.qr, self.kr, v, self.out, self.stats, self.dout, self.dq, self.dk, self.dv, *self.shape)
        c.rotary(self.dq, self.dq, self.dk, self.dk, self.B, self.L, self.H, self.Hkv, self.d, self.d, self.turns, flags=self.rinverse)

    def value(self):
        f = lambda x: x.numpy().astype(np.float64)
        return float((f(self.lp) * f(self.dlp)).sum() + (f(self.ent) * f(self.dent)).sum())

    def results(self):
        return [x.numpy() for x in (self.lp, self.ent, self.out, self.dq, self.dk, self.dv)]

    def release(self):
        for x in list(vars(self).values()):
            if hasattr(x, "release"):
                x.release()


def test_gradients_by_differences(ctx):
    """The slope along a random direction.  Central differences at h and 2 h, the h^2 term taken off: what is left of the
    difference quotient is O(h^4) of a fifth derivative, 2^-20 at h = 2^-5, and the outputs' own rounding, 2^-17 over h of values
    that add up to some hundreds; together below 1 % of the sum of the parts' sizes."""
    m, rng = Model(ctx), np.random.default_rng(22)
    q, k, v = _f32(rng, *m.qr.shape), _f32(rng, *m.kr.shape), _f32(rng, *m.kr.shape)
    uq, uk, uv = _f32(rng, *q.shape), _f32(rng, *k.shape), _f32(rng, *v.shape)

    def at(t):
        bufs = [ctx.to_device(x + np.float32(t) * u) for x, u in ((q, uq), (k, uk), (v, uv))]
        m.forward(*bufs)
        r = m.value()
        for b in bufs:
            b.release()
        return r

    h = 2.0 ** -5
    s1, s2 = (at(h) - at(-h)) / (2 * h), (at(2 * h) - at(-2 * h)) / (4 * h)
    slope = s1 + (s1 - s2) / 3
    bufs = [ctx.to_device(x) for x in (q, k, v)]
    m.forward(*bufs)
    m.backward(*bufs)
    parts = [float((g.numpy().astype(np.float64) * u).sum()) for g, u in ((m.dq, uq), (m.dk, uk), (m.dv, uv))]
    assert abs(slope - sum(parts)) <= 0.01 * sum(abs(p) for p in parts), (slope, parts)
    for b in bufs:
        b.release()
    m.release()


def test_a_training_step_recorded(ctx):
    from dl4s_amd import lib
    if not lib.graph_supported():
        pytest.skip("graph launches abort the queue under rocprofv3")
    m, rng = Model(ctx), np.random.default_rng(23)
    hosts = [[_f32(rng, *s) for s in (m.qr.shape, m.kr.shape, m.kr.shape)] for _ in range(4)]
    bufs = [ctx.to_device(x) for x in hosts[0]]
    m.forward(*bufs)
    m.backward(*bufs)
    ctx.graph_begin()
    m.forward(*bufs)
    m.backward(*bufs)
    graph = ctx.graph_end()
    for x in hosts:
        for b, h in zip(bufs, x):
            ctx.assign_h2d(b, h)
        m.forward(*bufs)                              # issued one by one, in between
        m.backward(*bufs)
        want = m.results()
        for o in (m.qr, m.kr, m.out, m.stats, m.logits, m.lp, m.ent, m.lstats, m.dlogits, m.dout, m.dq, m.dk, m.dv):
            ctx.fill(float("nan"), o, int(np.prod(o.shape)))
        ctx.sync()
        graph.replay()
        for a, b in zip(m.results(), want):
            assert np.array_equal(a, b)
    graph.destroy()
    for b in bufs:
        b.release()
    m.release()


def test_two_contexts_at_once():
    """Two streams, their calls interleaved without waiting: each gets what it gets alone."""
    from dl4s_amd import lib
    ctxs = [lib.Context(0) for _ in range(2)]
    models = [Model(c) for c in ctxs]
    rng = np.random.default_rng(24)
    ins = [[c.to_device(_f32(rng, *s)) for s in (m.qr.shape, m.kr.shape, m.kr.shape)] for c, m in zip(ctxs, models)]
    want = []
    for m, x in zip(models, ins):
        m.forward(*x)
        m.backward(*x)
        want.append(m.results())
    for _ in range(5):
        for m, x in zip(models, ins):
            m.forward(*x)
        for m, x in zip(models, ins):
            m.backward(*x)
    for m, w in zip(models, want):
        for a, b in zip(m.results(), w):
            assert np.array_equal(a, b)
    for c, m, x in zip(ctxs, models, ins):
        for b in x:
            b.release()
        m.release()
        c.close()


@pytest.mark.parametrize("recorded", [False, True])
@pytest.mark.parametrize("window,sinks", [(9, 0), (24, 3), (1000, 0)])
def test_a_prompt_and_the_steps_after_it(ctx, window, sinks, recorded):
    """A prompt through rotary_append and the forward pass over the cache, then one token after another by device positions and
    lengths: every row is the formula's over the rows that the cache holds then, and the keys in the cache are the bits
    that the rotary call gives for the whole sequence at once.  Recorded: one graph, replayed for every step."""
    from dl4s_amd import lib
    if recorded and not lib.graph_supported():
        pytest.skip("graph launches abort the queue under rocprofv3")
    B, H, Hkv, d, rot, prompt, steps, Tcap = 2, 6, 2, 40, 32, 21, 12, 40
    L, rng, rT = prompt + steps, np.random.default_rng(window), 0.15
    q, k, v = _f32(rng, B, H, L, d), _f32(rng, B, Hkv, L, d), _f32(rng, B, Hkv, L, d)
    turns = ctx.to_device(lib.rotary_frequencies(rot), np.float64)
    qa, ka, qt, kt = ctx.to_device(q), ctx.to_device(k), ctx.empty(q.shape), ctx.empty(k.shape)
    ctx.rotary(qa, qt, ka, kt, B, L, H, Hkv, d, rot, turns)
    q_turned, k_turned = qt.numpy(), kt.numpy()
    want = attention(q_turned, k_turned, v, rT, window, sinks)["out"]

    kc, vc = (ctx.to_device(np.full((B, Hkv, Tcap, d), np.nan)) for _ in range(2))
    bufs = [ctx.to_device(x[:, :, :prompt]) for x in (q, k, v)]
    qo, out = ctx.empty(bufs[0].shape), ctx.empty(bufs[0].shape)
    ctx.rotary_append(*bufs, qo, kc, vc, B, prompt, H, Hkv, Tcap, d, rot, turns)
    # the cache has room behind the prompt: lengths say what is valid
    lengths = ctx.to_device(np.full(B, prompt), np.int32)
    ctx.sdpa_window_fwd(qo, kc, vc, out, None, B, H, Hkv, prompt, Tcap, d, rT, ctx.window_desc(window, sinks, 0, lengths))
    assert_within(out.numpy(), (want[0][:, :, :prompt], want[1][:, :, :prompt]), "prompt")
    step = [ctx.empty((B, n, 1, d)) for n in (H, Hkv, Hkv)]
    q1, o1, position = ctx.empty((B, H, 1, d)), ctx.empty((B, H, 1, d)), ctx.to_device(np.full(B, prompt), np.int32)

    def one_step():
        ctx.rotary_append(*step, q1, kc, vc, B, 1, H, Hkv, Tcap, d, rot, turns, positions=position)
        ctx.sdpa_window_decode(q1, kc, vc, o1, B, H, Hkv, Tcap, Tcap, d, rT, window, sinks, lengths)

    graph = None
    for t in range(prompt, L):
        for b, x in zip(step, (q, k, v)):
            ctx.assign_h2d(b, x[:, :, t:t + 1])
        ctx.assign_h2d(position, np.full(B, t, np.int32))
        ctx.assign_h2d(lengths, np.full(B, t + 1, np.int32))
        if recorded and graph is None:
            one_step()                                     # (writes the rows that the first replay writes again)
            ctx.graph_begin()
            one_step()
            graph = ctx.graph_end()
        ctx.fill(float("nan"), o1, B * H * d)
        ctx.sync()
        graph.replay() if recorded else one_step()
        assert_within(o1.numpy(), (want[0][:, :, t:t + 1], want[1][:, :, t:t + 1]), "step %d" % t)
    assert np.array_equal(kc.numpy()[:, :, :L], k_turned) and np.array_equal(vc.numpy()[:, :, :L], v)
    assert np.isnan(kc.numpy()[:, :, L:]).all()
    if graph is not None:
        graph.destroy()
    for b in bufs + step + [turns, qa, ka, qt, kt, kc, vc, qo, out, lengths, q1, o1, position]:
        b.release()


def test_recording_needs_the_scratch_of_a_first_call(ctx):
    """A split decoding step and a split row of logits need the library's scratch block, which cannot grow while recording."""
    from dl4s_amd import lib
    if not lib.graph_supported():
        pytest.skip("graph launches abort the queue under rocprofv3")
    fresh = lib.Context(0)
    x, y, z = fresh.to_device(np.zeros((1, 1, 20000, 64))), fresh.to_device(np.zeros((1, 1, 1, 64))), fresh.empty((1, 1, 1, 64))
    t, lp = fresh.to_device(np.zeros(1), np.int32), fresh.empty((1,))
    calls = (lambda: fresh.sdpa_window_decode(y, x, x, z, 1, 1, 1, 20000, 20000, 64, 1.0, 20000),
             lambda: fresh.token_logprobs(x, 1, 1000000, 1000000, t, lp, top_k=0),
             lambda: fresh.sdpa_window_bwd(x, x, x, x, x, x, x, x, x, 1, 1, 1, 100, 100, 64, 1.0, fresh.window_desc(4)))
    fresh.graph_begin()
    for call in calls:
        with pytest.raises(lib.Dl4sHipError, match="run the same calls once before recording"):
            call()
    fresh.graph_end(keep=False)
    for b in (x, y, z, t, lp):
        b.release()
    fresh.close()


def test_an_inverse_temperature_of_zero_is_refused(ctx):
    from dl4s_amd import lib
    x = ctx.empty((64,))
    for t in (0.0, float("nan")):
        for call in (lambda: ctx.token_logprobs(x, 2, 16, 16, x, x, inv_temperature=t),
                     lambda: ctx.token_logprobs_bwd(x, 2, 16, 16, x, x, x, dlogprobs=x, inv_temperature=t)):
            with pytest.raises(lib.Dl4sHipError) as e:
                call()
            assert e.value.code == -1
    x.release()


@pytest.mark.parametrize("t", [-1.0, -0.3, 2.0 ** -30, 50.0])
def test_temperatures_of_the_log_probabilities(ctx, t):
    """Negative ones turn the order round; z = x t rounds once, here as in the operator, and the sums are off by a few steps."""
    rng = np.random.default_rng(25)
    rows, n = 3, 5001
    x = _f32(rng, rows, n)
    z = (x * np.float32(t)).astype(np.float64)
    e = np.exp(z - z.max(1, keepdims=True))
    lp = z - z.max(1, keepdims=True) - np.log(e.sum(1, keepdims=True))
    targets = np.array([0, 17, n - 1])
    bufs = [ctx.to_device(x), ctx.to_device(targets, np.int32), ctx.empty((rows,)), ctx.empty((rows, 4)), ctx.empty((rows, 4), np.int32)]
    ctx.token_logprobs(bufs[0], rows, n, n, bufs[1], bufs[2], inv_temperature=t, top_k=4, top_logprobs=bufs[3], top_tokens=bufs[4])
    order = np.argsort(-z, 1, kind="stable")[:, :4]
    assert np.array_equal(bufs[4].numpy(), order)
    spread = z.max() - z.min()
    bound = 2.0 ** -24 * (n / 64 + 100 + 8 * (1 + spread))
    assert np.abs(bufs[3].numpy() - np.take_along_axis(lp, order, 1)).max() <= bound
    assert np.abs(bufs[2].numpy() - lp[np.arange(rows), targets]).max() <= bound
    for b in bufs:
        b.release()


@pytest.mark.parametrize("rows,n", [(70000, 5), (131071, 3)])
def test_more_rows_than_a_grid_axis(ctx, rows, n):
    """Log probabilities and their gradient: the rows behind the 65535th are like the first ones, which are checked elsewhere."""
    rng = np.random.default_rng(26)
    first = 50
    x = np.resize(_f32(rng, first, n), (rows, n))
    targets, up = np.resize(rng.integers(0, n, first), rows), np.resize(_f32(rng, first), rows)
    got = []
    for m in (first, rows):
        bufs = [ctx.to_device(x[:m]), ctx.to_device(targets[:m], np.int32), ctx.to_device(up[:m])]
        outs = [ctx.empty((m,)), ctx.empty((m,)), ctx.empty((m, 3)), ctx.empty((m, 2)), ctx.empty((m, 2), np.int32), ctx.empty((m, n))]
        ctx.token_logprobs(bufs[0], m, n, n, bufs[1], outs[0], entropy=outs[1], stats=outs[2], top_k=2, top_logprobs=outs[3], top_tokens=outs[4])
        ctx.token_logprobs_bwd(bufs[0], m, n, n, bufs[1], outs[2], outs[5], dlogprobs=bufs[2], dentropy=bufs[2])
        got.append([o.numpy() for o in outs])
        for b in bufs + outs:
            b.release()
    # 16 wavefronts to a row for few rows, four for many: both end with the same one value a lane, in other lanes
    for a, b in zip(*got):
        a = np.resize(a, b.shape)
        assert np.array_equal(a, b) if a.dtype == np.int32 else np.abs(a - b).max() <= 2.0 ** -24 * 64 * (1 + np.abs(a).max())
