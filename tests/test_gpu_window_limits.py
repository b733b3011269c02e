"""Extents of the windowed attention's gradient that only the key side has: no query heads."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from dl4s_amd import lib
    c = lib.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("B,Hkv,Lk", [(1 << 29, 1 << 30, 1 << 29), (1, 1 << 31, 1), (1 << 20, 1 << 40, 1 << 10), (1 << 28, 8, 1)])
def test_key_heads_without_query_heads_are_limited_too(ctx, B, Hkv, Lk):
    """2^30 (batch, key head) pairs and more, some of which hold a number of rows that does not fit 64 bits."""
    from dl4s_amd import lib
    x = ctx.empty((64,))
    with pytest.raises(lib.Dl4sHipError) as e:
        ctx.sdpa_window_bwd(x, x, x, x, x, x, x, x, x, B, 0, Hkv, 5, Lk, 16, 1.0, ctx.window_desc(4))
    assert e.value.code == -5
    x.release()


def test_no_query_heads(ctx):
    """Nothing flows into the keys."""
    n = 3 * 2 * 7 * 16
    x, dk, dv = ctx.to_device(np.ones(n)), ctx.to_device(np.full(n + 5, np.nan)), ctx.to_device(np.full(n + 5, np.nan))
    ctx.sdpa_window_bwd(x, x, x, x, x, x, x, dk, dv, 3, 0, 2, 5, 7, 16, 1.0, ctx.window_desc(4))
    for b in (dk, dv):
        y = b.numpy()
        assert not y[:n].any() and np.isnan(y[n:]).all()
    for b in (x, dk, dv):
        b.release()
