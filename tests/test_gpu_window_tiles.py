"""The tiled kernels of the windowed attention - launches too large for the kernel that takes few rows - over head dims, layouts,
alignments, lengths, magnitudes and masked places, with four and with eight wavefronts to a workgroup's rows.  Bounds:
window_reference."""
import numpy as np
import pytest

from test_gpu_window_edges import _compare, _forward_backward, _inputs
from window_reference import assert_within, attention

pytestmark = pytest.mark.gpu

# (B, H, Hkv, L, window, sinks): the first two in small workgroups, the last with eight wavefronts a workgroup
SHAPES = [(14, 4, 2, 150, 40, 5), (33, 3, 3, 71, 33, 0), (9, 4, 2, 261, 200, 3)]


@pytest.fixture(scope="module")
def ctx():
    from dl4s_amd import lib
    c = lib.Context(0)
    yield c
    c.close()


def _scale(d):
    return float(np.float32(1 / np.sqrt(d)))


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("d", [1, 7, 16, 31, 32, 36, 50, 64, 65, 92, 96, 100, 127, 128])
def test_head_dims(ctx, d, shape):
    B, H, Hkv, L, window, sinks = shape
    q, k, v, g = _inputs(np.random.default_rng(d), B, H, Hkv, L, L, d)
    _compare(_forward_backward(ctx, q, k, v, g, _scale(d), window, sinks), attention(q, k, v, _scale(d), window, sinks, dout=g), "d %d" % d)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("sq,sk,sv,sg", [
    (2.0 ** -70, 2.0 ** 70, 1, 1), (2.0 ** 90, 2.0 ** -90, 1, 1), (1, 1, 2.0 ** -90, 2.0 ** 60), (1, 1, 2.0 ** 90, 2.0 ** -60),
    (4, 4, 1, 1), (0, 1, 1, 1), (1, 1, 0, 1)])
def test_magnitudes(ctx, sq, sk, sv, sg, shape):
    B, H, Hkv, L, window, sinks = shape
    for d in (64, 128):
        q, k, v, g = (x * np.float32(s) for x, s in zip(_inputs(np.random.default_rng(d), B, H, Hkv, L, L, d), (sq, sk, sv, sg)))
        want = attention(q, k, v, _scale(d), window, sinks, dout=g)
        _compare(_forward_backward(ctx, q, k, v, g, _scale(d), window, sinks), want, "scales %g %g %g %g" % (sq, sk, sv, sg))


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("d", [64, 96])
def test_masked_places(ctx, d, shape):
    """Lengths of all kinds; keys behind them, before every window and behind every query hold NaN and infinities, and so do
    the queries that see nothing."""
    B, H, Hkv, L, window, sinks = shape
    rng = np.random.default_rng(d)
    Lk, offset = L + 90, 60
    q, k, v, g = _inputs(rng, B, H, Hkv, L, Lk, d)
    lengths = rng.integers(-3, Lk + 5, B)
    lengths[:4] = Lk, 0, 1, 40
    want = attention(q, k, v, _scale(d), window, sinks, offset, lengths, g)
    hidden = np.r_[sinks:max(sinks, offset - window + 1), offset + L:Lk]
    k[:, :, hidden], v[:, :, hidden] = np.inf, np.nan
    for b, n in enumerate(lengths):
        n = max(0, min(n, Lk))
        k[b, :, n:], v[b, :, n:] = np.nan, np.inf
        seen = offset + np.arange(L) - window + 1 < n
        if min(n, sinks) > 0:
            seen[:] = True
        q[b, :, ~seen], g[b, :, ~seen] = np.nan, np.inf
    _compare(_forward_backward(ctx, q, k, v, g, _scale(d), window, sinks, offset, lengths), want, "masked places")


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("d", [64, 128])
def test_rows_of_unlike_sizes(ctx, d, shape):
    B, H, Hkv, L, window, sinks = shape
    rng = np.random.default_rng(d)
    q, k, v, g = (x * np.exp2(rng.integers(-4, 5, x.shape[:3] + (1,))).astype(np.float32) for x in _inputs(rng, B, H, Hkv, L, L, d))
    _compare(_forward_backward(ctx, q, k, v, g, 1 / 32.0, window, sinks), attention(q, k, v, 1 / 32.0, window, sinks, dout=g), "unlike rows")


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("d,shift", [(64, 0), (64, 1), (60, 2), (128, 3), (33, 0)])
def test_token_major_and_unaligned(ctx, d, shift, shape):
    """[B, L, heads, d] tensors that start `shift` floats off the 16-byte grid; what lies around the outputs stays."""
    from dl4s_amd import lib
    B, H, Hkv, L, window, sinks = shape
    q, k, v, g = _inputs(np.random.default_rng(d), B, H, Hkv, L, L, d)
    want = attention(q, k, v, _scale(d), window, sinks, dout=g)
    around = np.full(shift, 77.0, np.float32)
    lay = lambda x: np.concatenate([around, x.transpose(0, 2, 1, 3).ravel(), around])
    bufs = [ctx.to_device(lay(x)) for x in (q, k, v, g)]
    outs = [ctx.to_device(lay(np.full_like(x, np.nan))) for x in (q, q, k, k)]
    stats = ctx.empty((B, H, L, 2))
    iq, ik, iv, ig = (b.offset(4 * shift) for b in bufs)
    o, dq, dk, dv = (b.offset(4 * shift) for b in outs)
    args = (B, H, Hkv, L, L, d, _scale(d), ctx.window_desc(window, sinks), lib.SDPA_TOKEN_MAJOR)
    ctx.sdpa_window_fwd(iq, ik, iv, o, stats, *args)
    ctx.sdpa_window_bwd(iq, ik, iv, o, stats, ig, dq, dk, dv, *args)
    for name, b, like in zip(("out", "dq", "dk", "dv"), outs, (q, q, k, k)):
        x = b.numpy()
        assert (x[:shift] == 77).all() and (x[len(x) - shift:] == 77).all()
        x = x[shift:len(x) - shift].reshape(like.transpose(0, 2, 1, 3).shape).transpose(0, 2, 1, 3)
        assert_within(x, want[name], "shift %d %s" % (shift, name))
    for b in bufs + outs + [stats]:
        b.release()


def test_a_value_that_is_not_a_number_reaches_the_rows_that_see_it(ctx):
    q, k, v, g = _inputs(np.random.default_rng(5), 20, 2, 2, 200, 200, 64)
    q[3, 1, 77] = np.nan
    k[4, 0, 50] = np.nan
    out = _forward_backward(ctx, q, k, v, g, 0.125, 30)["out"]
    bad = np.zeros(out.shape[:3], bool)
    bad[3, 1, 77] = bad[4, 0, 50:80] = True
    assert np.isnan(out[bad]).all() and np.isfinite(out[~bad]).all()


@pytest.mark.parametrize("Lq,Lk", [(0, 5), (5, 0)])
@pytest.mark.parametrize("d", [16, 140])
def test_gradients_of_nothing(ctx, Lq, Lk, d):
    """No queries: zeros for the keys; no keys: zeros for the queries."""
    n = 2 * 5 * d
    x, stats = ctx.to_device(np.ones(n)), ctx.empty((2, 5, 2))
    out, dq, dk, dv = (ctx.to_device(np.full(n, np.nan)) for _ in range(4))
    args = (1, 2, 2, Lq, Lk, d, 1.0, ctx.window_desc(3))
    ctx.sdpa_window_fwd(x, x, x, out, stats, *args)
    ctx.sdpa_window_bwd(x, x, x, out, stats, x, dq, dk, dv, *args)
    for b, rows in ((out, Lq), (dq, Lq), (dk, Lk), (dv, Lk)):
        y = b.numpy()
        assert not y[:2 * rows * d].any() and np.isnan(y[2 * rows * d:]).all()
    for b in (x, stats, out, dq, dk, dv):
        b.release()
