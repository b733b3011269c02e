"""Log probabilities of given tokens, entropy, best alternatives and the gradient of the logits
(dl4s_hip_token_logprobs_f32, dl4s_hip_token_logprobs_bwd_f32) against the formulas in 64 bits.

Bounds, with u = 2^-24, z = x * t rounded once in both (the operator's definition), Y = max |z - m| over the row's tokens
that weigh anything: exp is off by 4 u (1 + |z - m|) of its value, a sum of n positive terms by n u at worst - here every
sum runs over lanes and pieces, at most n / 64 + 80 terms one behind the other - so
  l is off by e_l = u (n / 64 + 100 + 4 (1 + Y)) of its value, a log probability by e_l + 4 u (1 + |log p|),
  the entropy by 2 e_l (1 + Y) + 8 u (1 + entropy)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    from dl4s_amd import lib
    c = lib.Context(0)
    yield c
    c.close()


def _reference(x, t, targets, ignore):
    z32 = (x * np.float32(t)).astype(np.float32) + np.float32(0)
    z = z32.astype(np.float64)
    with np.errstate(all="ignore"):
        m = z.max(1, keepdims=True)
        e = np.exp(z - m)
        l = e.sum(1, keepdims=True)
        lp = z - m - np.log(l)
        p = e / l
        H = -np.where(p > 0, p * lp, 0).sum(1)
        Y = np.where(p > 1e-40, np.abs(z - m), 0).max(1)
    n = x.shape[1]
    e_l = U * (n / 64 + 100 + 4 * (1 + Y))
    at = np.clip(targets, 0, n - 1)
    got = lp[np.arange(len(x)), at]
    got = np.where(targets == ignore, 0.0, np.where((targets < 0) | (targets >= n), np.nan, got))
    return z32, z, lp, p, H, Y, e_l, got


def _close(got, want, bound, what):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    with np.errstate(all="ignore"):
        ok = (np.abs(got - want) <= bound) | (np.isnan(got) & np.isnan(want)) | (got == want)
    assert ok.all(), "%s: %d of %d outside, got %s want %s" % (what, (~ok).sum(), ok.size, got[~ok][:4], want[~ok][:4])


def _order(z32, k):
    """Tokens by falling z, equal ones by rising token, NaN last."""
    key = np.where(np.isnan(z32), -np.inf, z32.astype(np.float64))
    return np.lexsort((np.broadcast_to(np.arange(z32.shape[1]), z32.shape), np.isnan(z32), -key), axis=1)[:, :k]


def _check(ctx, x, n, t=1.0, targets=None, ignore=-1, top=0, entropy=True, grads=False, what="", inplace=False):
    rows, stride = x.shape
    rng = np.random.default_rng(rows + n)
    if targets is None:
        targets = rng.integers(0, n, rows)
    z32, z, lp, p, H, Y, e_l, want = _reference(x[:, :n], t, targets, ignore)
    dx, dt = ctx.to_device(x), ctx.to_device(targets, np.int32)
    o = {s: ctx.to_device(np.full(shape, np.nan)) for s, shape in (("lp", (rows,)), ("H", (rows,)), ("stats", (rows, 3)),
                                                                  ("top", (rows, max(top, 1))))}
    ids = ctx.to_device(np.full((rows, max(top, 1)), -7), np.int32)
    ctx.token_logprobs(dx, rows, n, stride, dt, o["lp"], entropy=o["H"] if entropy else None, stats=o["stats"], inv_temperature=t,
                       ignore_index=ignore, top_k=top, top_logprobs=o["top"] if top else None, top_tokens=ids if top else None)
    with np.errstate(all="ignore"):
        _close(o["lp"].numpy(), want, e_l + 4 * U * (1 + np.abs(want)), what + " log probability")
        if entropy:
            _close(o["H"].numpy(), H, 2 * e_l * (1 + Y) + 8 * U * (1 + np.abs(H)), what + " entropy")
        if top:
            order = _order(z32, top)
            assert np.array_equal(ids.numpy(), order), what + " alternatives"
            best = np.take_along_axis(lp, order, 1)
            _close(o["top"].numpy(), best, e_l[:, None] + 4 * U * (1 + np.abs(best)), what + " alternatives' log probabilities")
        if grads:
            g, h = (rng.standard_normal(rows).astype(np.float32) for _ in range(2))
            d_g, d_h = ctx.to_device(g), ctx.to_device(h)
            e_p = e_l[:, None] + 8 * U * (1 + np.abs(lp))                # of a probability, relative
            for use_g, use_h in ((True, True), (True, False), (False, True), (False, False)):
                a = np.where(targets == ignore, 0, np.where((targets < 0) | (targets >= n), np.nan, g.astype(np.float64)))[:, None]
                a, b = a if use_g else 0 * g[:, None], h.astype(np.float64)[:, None] * use_h
                hit = np.arange(n)[None] == targets[:, None]
                lph = np.where(p > 0, lp + H[:, None], 0)
                d = np.where(hit, a, 0) - p * a - b * p * lph
                bound = 4 * U * np.abs(a) * hit + p * np.abs(a) * (e_p + 8 * U) + np.abs(b) * p * (
                    np.abs(lph) * (e_p + 8 * U) + 3 * e_l[:, None] * (1 + Y[:, None]) + 16 * U * (1 + np.abs(lph)))
                out = ctx.to_device(np.full((rows, stride), 123.0)) if not inplace else ctx.to_device(x)
                ctx.token_logprobs_bwd(out if inplace else dx, rows, n, stride, dt, o["stats"], out, dlogprobs=d_g if use_g else None,
                                       dentropy=d_h if use_h else None, inv_temperature=t, ignore_index=ignore)
                got = out.numpy()
                _close(got[:, :n], d * float(np.float32(t)), bound * abs(t) + 1e-43, what + " gradient")
                assert np.array_equal(got[:, n:], x[:, n:] if inplace else np.full((rows, stride - n), 123.0, np.float32), equal_nan=True)
                out.release()
            d_g.release()
            d_h.release()
    for b in list(o.values()) + [dx, dt, ids]:
        b.release()


SIZES = [(1, 1, 1), (3, 2, 2), (1, 63, 63), (2, 64, 70), (5, 65, 65), (1, 255, 256), (7, 1000, 1001), (2, 1024, 1024), (3, 4097, 4100),
         (300, 50, 51), (2, 32000, 32000), (1, 50257, 50304), (33, 5003, 5003), (1, 150001, 150001), (2000, 7, 7), (9, 16384, 16384)]


@pytest.mark.parametrize("rows,n,stride", SIZES)
def test_sizes(ctx, rows, n, stride):
    rng = np.random.default_rng(rows * n)
    x = (rng.standard_normal((rows, stride)) * 3).astype(np.float32)
    x[:, n:] = np.nan                                        # what stands between the rows is never used
    targets = rng.integers(0, n, rows)
    targets[::3] = -1
    _check(ctx, x, n, targets=targets, top=min(n, 10), grads=True, what="%d x %d" % (rows, n))
    _check(ctx, x, n, t=0.37, targets=targets, top=min(n, 64), grads=True, what="%d x %d t" % (rows, n), inplace=True)
    _check(ctx, x, n, t=1.9, top=min(n, 1), entropy=False, what="%d x %d no entropy" % (rows, n))


@pytest.mark.parametrize("n", [64, 1000, 9000, 70000])
@pytest.mark.parametrize("kind", ["equal", "two values", "rising", "falling", "zeros of both signs", "coarse", "blocked", "one left",
                                  "late maximum"])
def test_orders_and_ties(ctx, n, kind):
    rng = np.random.default_rng(n)
    x = rng.standard_normal((3, n)).astype(np.float32)
    if kind == "equal":
        x[:] = 0.75
    elif kind == "two values":
        x[:] = (rng.random((3, n)) < 0.01)
    elif kind == "rising":
        x[:] = np.linspace(-30, 30, n)
    elif kind == "falling":
        x[:] = np.linspace(30, -30, n)
    elif kind == "zeros of both signs":
        x[:] = np.where(rng.random((3, n)) < 0.5, 0.0, -0.0)
    elif kind == "coarse":
        x[:] = np.round(x * 2)
    elif kind == "blocked":
        x[:, rng.random(n) < 0.9] = -np.inf
        x[:, :3] = -np.inf
        x[:, 5] = 1.0
    elif kind == "one left":
        x[:] = -np.inf
        x[:, n // 2] = 3.0
    elif kind == "late maximum":
        x[:, -1] = 200.0
    targets = np.array([0, n - 1, n // 2])
    for top in (1, 20, 64):
        _check(ctx, x, n, targets=targets, top=top, grads=top == 1, what=kind)


def test_targets_outside(ctx):
    x = np.random.default_rng(0).standard_normal((6, 100)).astype(np.float32)
    _check(ctx, x, 100, targets=np.array([-1, 100, 5, -100, 2 ** 31 - 1, 99]), ignore=-100, top=3, grads=True, what="outside")


def test_not_a_number(ctx):
    """A NaN makes its row's sums NaN and comes last in the order; a row of nothing but -inf has no distribution."""
    x = np.random.default_rng(1).standard_normal((4, 300)).astype(np.float32)
    x[0, 7] = np.nan
    x[1] = -np.inf
    x[2, 9] = np.inf
    dx, dt = ctx.to_device(x), ctx.to_device(np.array([3, 3, 3, 3]), np.int32)
    lp, H, top, ids = ctx.empty((4,)), ctx.empty((4,)), ctx.empty((4, 64)), ctx.empty((4, 64), np.int32)
    ctx.token_logprobs(dx, 4, 300, 300, dt, lp, entropy=H, top_k=64, top_logprobs=top, top_tokens=ids)
    assert np.isnan(lp.numpy()).tolist() == [True, True, True, False]
    assert np.isnan(H.numpy()).tolist() == [True, True, True, False]
    assert np.array_equal(ids.numpy(), _order(x, 64))
    for b in (dx, dt, lp, H, top, ids):
        b.release()


def test_one_token_after_another_gives_the_same_bits(ctx):
    """Two calls, the same bits: the merge of a split row does not depend on which piece was ready first."""
    rng = np.random.default_rng(3)
    x = ctx.to_device((rng.standard_normal((2, 60001)) * 2).astype(np.float32))
    t = ctx.to_device(np.array([5, 60000]), np.int32)
    a = [ctx.empty((2,)) for _ in range(4)]
    ctx.token_logprobs(x, 2, 60001, 60001, t, a[0], entropy=a[1])
    ctx.token_logprobs(x, 2, 60001, 60001, t, a[2], entropy=a[3])
    assert np.array_equal(a[0].numpy(), a[2].numpy()) and np.array_equal(a[1].numpy(), a[3].numpy())
    for b in a + [x, t]:
        b.release()


def test_offsets_past_32_bits(ctx):
    """Rows that lie more than 2^31 floats behind the first one."""
    rows, n, stride = 3, 1000, (1 << 30) + 8
    rng = np.random.default_rng(5)
    x = rng.standard_normal((rows, n)).astype(np.float32)
    big = ctx.empty(((rows - 1) * stride + n,))
    for r in range(rows):
        part = ctx.to_device(x[r])
        from dl4s_amd import lib
        import ctypes as C
        lib._check(ctx.lib.dl4s_hip_assign_d2d(ctx.handle, C.c_void_p(big.offset(4 * r * stride)), C.c_void_p(part.ptr), C.c_size_t(4 * n)))
        part.release()
    t, lp, ids, top = ctx.to_device(np.array([1, 2, 3]), np.int32), ctx.empty((rows,)), ctx.empty((rows, 5), np.int32), ctx.empty((rows, 5))
    ctx.token_logprobs(big, rows, n, stride, t, lp, top_k=5, top_logprobs=top, top_tokens=ids)
    _, _, lps, _, _, _, e_l, want = _reference(x, 1.0, np.array([1, 2, 3]), -1)
    _close(lp.numpy(), want, e_l + 4 * U * (1 + np.abs(want)), "far rows")
    assert np.array_equal(ids.numpy(), _order(x, 5))
    for b in (big, t, lp, ids, top):
        b.release()
    ctx.pool_trim(0)


def test_unaligned_rows(ctx):
    rng = np.random.default_rng(6)
    for off in (1, 2, 3):
        x = rng.standard_normal((3, 5001)).astype(np.float32)
        d = ctx.to_device(np.concatenate([np.full(off, np.nan, np.float32), x.ravel()]))
        t, lp = ctx.to_device(np.array([0, 1, 5000]), np.int32), ctx.empty((3,))
        ids, top = ctx.empty((3, 9), np.int32), ctx.empty((3, 9))
        ctx.token_logprobs(d.offset(4 * off), 3, 5001, 5001, t, lp, top_k=9, top_logprobs=top, top_tokens=ids)
        _, _, _, _, _, _, e_l, want = _reference(x, 1.0, np.array([0, 1, 5000]), -1)
        _close(lp.numpy(), want, e_l + 4 * U * (1 + np.abs(want)), "unaligned")
        assert np.array_equal(ids.numpy(), _order(x, 9))
        for b in (d, t, lp, ids, top):
            b.release()


@pytest.mark.parametrize("change,code", [
    (dict(rows=-1), -1), (dict(n=0), -5), (dict(stride=9), -2), (dict(top_k=65, n=100, stride=100), -5), (dict(top_k=11), -2),
    (dict(top_k=-1), -5), (dict(null=True), -1), (dict(no_targets=True), -1), (dict(top_k=2, no_top=True), -1)])
def test_refusals(ctx, change, code):
    from dl4s_amd import lib
    a = dict(rows=2, n=10, stride=10, top_k=0, null=False, no_targets=False, no_top=False)
    a.update(change)
    x = ctx.empty((400,))
    with pytest.raises(lib.Dl4sHipError) as e:
        ctx.token_logprobs(None if a["null"] else x, a["rows"], a["n"], a["stride"], None if a["no_targets"] else x, x, top_k=a["top_k"],
                           top_logprobs=None if a["no_top"] else x, top_tokens=x)
    assert e.value.code == code
    x.release()


def test_gradient_refusals_and_empty_calls(ctx):
    from dl4s_amd import lib
    x = ctx.empty((400,))
    for kw, code in ((dict(stats=None), -1), (dict(dlogits=None), -1), (dict(targets=None), -1), (dict(n=0), -5), (dict(stride=9), -2)):
        a = dict(logits=x, n=10, stride=10, targets=x, stats=x, dlogits=x)
        a.update(kw)
        with pytest.raises(lib.Dl4sHipError) as e:
            ctx.token_logprobs_bwd(a["logits"], 2, a["n"], a["stride"], a["targets"], a["stats"], a["dlogits"], dlogprobs=x)
        assert e.value.code == code
    ctx.token_logprobs(None, 0, 10, 10, None, None)
    ctx.token_logprobs_bwd(None, 0, 10, 10, None, None, None)
    x.release()
