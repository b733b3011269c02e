"""Log probabilities of rows most of whose tokens are masked, with large finite values (the type's lowest among them) or with -inf.
Reference and bounds: test_gpu_token_logprobs."""
import numpy as np
import pytest

from test_gpu_token_logprobs import U, _check, _close, _reference

pytestmark = pytest.mark.gpu

LOWEST = float(np.finfo(np.float32).min)
# (rows, n): one row to 16 wavefronts; rows in parts; more rows than compute units, four wavefronts to a row
SHAPES = [(3, 1000), (2, 9001), (2, 70000), (600, 1300)]


@pytest.fixture(scope="module")
def ctx():
    from dl4s_amd import lib
    c = lib.Context(0)
    yield c
    c.close()


def _masked(rng, rows, n, mask, live):
    """Logits with `live` tokens that are not masked, the last one among them, and targets: a live token, in every fifth row a masked one."""
    x = np.full((rows, n), mask, np.float32)
    targets = np.empty(rows, np.int64)
    for r in range(rows):
        at = np.append(rng.choice(n - 1, live - 1, replace=False), n - 1)
        x[r, at] = rng.standard_normal(live) * 2
        targets[r] = at[rng.integers(live)]
        if r % 5 == 4:
            targets[r] = np.delete(np.arange(n), at)[rng.integers(n - live)]
    return x, targets


def _gradient(ctx, x, t, targets, ignore, g, h=None, spoil=False):
    """dlogits for upstream gradients g (log probabilities) and h (entropies); spoil: the entropies kept for it are NaN."""
    rows, n = x.shape
    bufs = [ctx.to_device(x), ctx.to_device(targets, np.int32), ctx.to_device(g)] + ([ctx.to_device(h)] if h is not None else [])
    lp, stats, out = ctx.empty((rows,)), ctx.empty((rows, 3)), ctx.to_device(np.full((rows, n), 123.0))
    ctx.token_logprobs(bufs[0], rows, n, n, bufs[1], lp, stats=stats, inv_temperature=t, ignore_index=ignore)
    if spoil:
        s = stats.numpy()
        s[:, 2] = np.nan
        ctx.assign_h2d(stats, s)
    ctx.token_logprobs_bwd(bufs[0], rows, n, n, bufs[1], stats, out, dlogprobs=bufs[2], dentropy=bufs[3] if h is not None else None,
                           inv_temperature=t, ignore_index=ignore)
    got = out.numpy()
    for b in bufs + [lp, stats, out]:
        b.release()
    return got


def _gradient_of_log_probabilities(x, t, targets, g):
    """Value and bound of (1[j = target] - p) g t, the bound as in test_gpu_token_logprobs with no entropy term."""
    _, _, lp, p, _, _, e_l, _ = _reference(x, t, targets, -1)
    a, hit = g.astype(np.float64)[:, None], np.arange(x.shape[1])[None] == targets[:, None]
    e_p = e_l[:, None] + 8 * U * (1 + np.where(p > 0, np.abs(lp), 0))
    d = (np.where(hit, a, 0) - p * a) * float(np.float32(t))
    return d, abs(t) * (4 * U * np.abs(a) * hit + p * np.abs(a) * (e_p + 8 * U)) + 1e-43


@pytest.mark.parametrize("rows,n", SHAPES)
@pytest.mark.parametrize("mask", [LOWEST, -1e37, -1e9, -np.inf])
def test_gradient_without_the_entropy(ctx, mask, rows, n):
    """A loss of log probabilities alone: the gradient of masked rows, whatever their entropy came to."""
    rng = np.random.default_rng(n)
    x, targets = _masked(rng, rows, n, mask, 8)
    if np.isinf(mask):
        targets = np.full(rows, n - 1)                      # (a blocked token's log probability is -inf)
    g = rng.standard_normal(rows).astype(np.float32)
    d, bound = _gradient_of_log_probabilities(x, 1.0, targets, g)
    for spoil in (False, True):
        _close(_gradient(ctx, x, 1.0, targets, -1, g, spoil=spoil), d, bound, "gradient")
    # an upstream gradient of zero for the entropies is the same as none
    _close(_gradient(ctx, x, 1.0, targets, -1, g, h=np.zeros(rows)), d, bound, "gradient, entropies' zero")


@pytest.mark.parametrize("rows,n", SHAPES)
@pytest.mark.parametrize("top", [0, 20])
@pytest.mark.parametrize("mask", [LOWEST, -1e38, -1e37, -1e36, -1e9])
def test_entropies_of_masked_rows(ctx, mask, top, rows, n):
    """A lane, a wavefront or a part of a row may meet nothing but masked tokens: their distance to the row's maximum, times
    their number, is past fp32's range where their weight is zero."""
    rng = np.random.default_rng(n + top)
    for live, t in ((8, 1.0), (1, 0.7)):
        x, targets = _masked(rng, rows, n, mask, live)
        _check(ctx, x, n, t=t, targets=targets, top=top, grads=True, what="mask %g, %d live" % (mask, live))
    x, targets = _masked(rng, rows, n, mask, n // 2)
    _check(ctx, x, n, targets=targets, top=top, grads=True, what="mask %g, half" % mask)


@pytest.mark.parametrize("n", [700, 40000])
def test_logits_from_end_to_end_of_the_range(ctx, n):
    """Rows whose logits rise or fall over the whole range of fp32, and rows of nothing but its lowest value."""
    x = np.empty((4, n), np.float32)
    x[0] = np.linspace(LOWEST, -LOWEST, n)
    x[1] = x[0, ::-1]
    x[2] = LOWEST
    x[3] = np.where(np.arange(n) % 2, LOWEST, 0.0)
    for top in (0, 7):
        _check(ctx, x, n, targets=np.array([n - 1, 0, n // 2, 2]), top=top, grads=True, what="range")


@pytest.mark.parametrize("n", [1, 63, 1000, 5001, 9000])
def test_ignored_rows_of_blocked_tokens(ctx, n):
    """Padding: every logit -inf, or NaN, the target ignored.  Nothing flows back into such a row, and its log probability is zero."""
    rng = np.random.default_rng(n)
    rows = 6
    x = rng.standard_normal((rows, n)).astype(np.float32)
    targets, g, h = rng.integers(0, n, rows), rng.standard_normal(rows).astype(np.float32), np.zeros(rows, np.float32)
    x[1], x[3], x[4] = -np.inf, np.nan, np.inf
    targets[[1, 3, 4, 5]] = -1
    d, bound = _gradient_of_log_probabilities(x[[0, 2]], 0.9, targets[[0, 2]], g[[0, 2]])
    for up in (None, h):
        got = _gradient(ctx, x, 0.9, targets, -1, g, h=up)
        assert not got[[1, 3, 4, 5]].any(), "padding rows"
        _close(got[[0, 2]], d, bound, "rows between padding")


def test_rows_that_no_gradient_reaches(ctx):
    """An upstream gradient of zero is no gradient, in rows with targets too; a target outside the vocabulary stays NaN."""
    x = np.random.default_rng(2).standard_normal((4, 300)).astype(np.float32)
    x[0], x[3] = -np.inf, -np.inf
    targets = np.array([5, 5, 300, 7])
    got = _gradient(ctx, x, 1.0, targets, -1, np.array([0, 0, 0, 1.0], np.float32))
    assert not got[:2].any() and np.isnan(got[2]).all() and np.isnan(got[3]).all()
