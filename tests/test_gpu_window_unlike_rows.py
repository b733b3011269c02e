"""Windowed attention of tensors whose rows differ in size by more than 2^13: a row that is read long after, or in another head than,
a larger one is as exact as if that one were not there.

The outputs compared are those that no large row enters.  Their exact values are the same with the large rows replaced by zeros, and
the bounds (window_reference) are those of the tensors with the large rows replaced: nothing in them knows of the large rows."""
import numpy as np
import pytest

from test_gpu_window_edges import _forward_backward, _inputs
from window_reference import assert_within, attention

pytestmark = pytest.mark.gpu

SPREADS = [8, 16, 20, 30, 60]
# (B, H, Hkv, L, window): in the first two four wavefronts have a workgroup's rows for themselves, in the last two eight share them;
# every one is too large for the kernel that takes few rows
SHAPES = [(14, 4, 2, 230, 32), (40, 2, 2, 210, 20), (9, 4, 2, 461, 200), (8, 8, 8, 500, 220)]


@pytest.fixture(scope="module")
def ctx():
    from dl4s_amd import lib
    c = lib.Context(0)
    yield c
    c.close()


def _scale(d):
    return float(np.float32(1 / np.sqrt(d)))


def _ends(*tensors):
    """The first and the last batch element, which are compared."""
    return [x[[0, -1]] for x in tensors]


def _compare(got, want, names, rows, what):
    for name in names:
        value, bound = (x[:, :, rows] for x in want[name])
        assert_within(got[name][[0, -1]][:, :, rows], (value, bound), "%s of %s" % (name, what))


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("r", SPREADS)
@pytest.mark.parametrize("which", ["q", "k", "v", "dout"])
def test_rows_behind_larger_ones(ctx, which, r, d, shape):
    """The first 64 rows of one tensor are of size one, the others of size 2^-r: results of what sees only the others.  Where that
    would make the scores tiny, the other factor is 2^r times as large for the rows that meet only small ones."""
    B, H, Hkv, L, window = shape
    tensors = dict(zip(("q", "k", "v", "dout"), _inputs(np.random.default_rng(r + d), B, H, Hkv, L, L, d)))
    tensors[which][:, :, 64:] *= np.float32(2.0 ** -r)
    if which == "q":
        tensors["k"][:, :, 64:] *= np.float32(2.0 ** r)     # seen by queries from 64 on
    if which == "k":
        tensors["q"][:, :, 64 + window:] *= np.float32(2.0 ** r)        # see keys from 65 on
    got = _forward_backward(ctx, *tensors.values(), _scale(d), window)
    tensors[which][:, :, :64] = 0
    q, k, v, g = _ends(*tensors.values())
    want = attention(q, k, v, _scale(d), window, dout=g)
    # rows from 64 + window on neither see the first 64 nor are seen by them
    _compare(got, want, ("dq", "dk", "dv") + (("out",) if which != "v" else ()), slice(64 + window, L), "rows behind larger " + which)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("r", SPREADS + [-30])
def test_outputs_behind_larger_values(ctx, r, d, shape):
    """Queries of one wavefront, some of which see values 2^r times as large as all the others'."""
    B, H, Hkv, L, window = shape
    q, k, v, g = _inputs(np.random.default_rng(r + d + 200), B, H, Hkv, L, L, d)
    at = slice(32, 64)
    v[:, :, at] *= np.float32(2.0 ** r)
    got = _forward_backward(ctx, q, k, v, g, _scale(d), window)
    v[:, :, at] = 0
    want = attention(*_ends(q, k, v), _scale(d), window)
    for rows in (slice(0, 32), slice(63 + window, L)):
        _compare(got, want, ["out"], rows, "rows beside larger values")


@pytest.mark.parametrize("sizes", [(2.0 ** 110, 2.0 ** -60, 1.0), (2.0 ** -110, 2.0 ** 100, 2.0 ** -90)])
@pytest.mark.parametrize("shape", SHAPES[:3:2])
@pytest.mark.parametrize("d", [64, 128])
def test_values_of_all_sizes(ctx, d, shape, sizes):
    """Neighbouring tiles at opposite ends of the range of fp32: no sum leaves it, and a row that sees only one of the sizes has that
    size's precision within 2^-60 of the largest."""
    B, H, Hkv, L, window = shape
    window = 16
    q, k, v, g = _inputs(np.random.default_rng(d), B, H, Hkv, L, L, d)
    step = np.arange(L) // 64 % 3
    v *= np.asarray(sizes, np.float32)[step][None, None, :, None]
    out = _forward_backward(ctx, q, k, v, g, _scale(d), window)["out"]
    assert np.isfinite(out).all()
    for n, size in enumerate(sizes):
        part = np.where((step == n)[None, None, :, None], v, 0)
        value, bound = attention(*_ends(q, k, part), _scale(d), window)["out"]
        rows = (step == n) & (np.arange(L) % 64 >= window) & (np.arange(L) >= window)
        # beside the bound: each of the window's weights off by half a step of its low plane, 2^-25, times planes of up to 2^15, in units
        # of 2^-60 of those that hold the largest value (below 8 sizes, and 2^11 units or more), over a sum of weights of 2^7 or more
        beside = window * 2.0 ** (-25 + 15 - 60 - 11 - 7) * 8 * max(sizes)
        assert_within(out[[0, -1]][:, :, rows], (value[:, :, rows], bound[:, :, rows] + beside), "size %g" % size)


@pytest.mark.parametrize("r", SPREADS)
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("B,H,Hkv,L,window", [(2, 4, 1, 200, 8), (20, 8, 4, 200, 8), (3, 6, 2, 300, 8)])
def test_shared_heads_beside_larger_rows(ctx, r, d, B, H, Hkv, L, window):
    """Query heads of a group, one after the other: rows that some keys of a wavefront see are larger in every head, and the sums
    of the keys that do not see them go on in the next head as exactly as they began."""
    at = slice(32, 64)
    for which in (0, 3):                                    # q: dk; dout: dk and dv
        tensors = _inputs(np.random.default_rng(r + d + 300), B, H, Hkv, L, L, d)
        large = tensors[which][:, :, at].copy()
        tensors[which] *= np.float32(2.0 ** -r)
        tensors[which][:, :, at] = large
        got = _forward_backward(ctx, *tensors, _scale(d), window)
        tensors[which][:, :, at] = 0
        q, k, v, g = _ends(*tensors)
        want = attention(q, k, v, _scale(d), window, dout=g)
        for keys in (slice(0, 25), slice(64, L)):           # key 24 is seen up to row 31, key 64 from row 64 on
            _compare(got, want, ("dk", "dv"), keys, "shared heads")


@pytest.mark.parametrize("r", SPREADS)
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("B,H,Hkv,L,window", [(2, 2, 2, 300, 70), (24, 4, 2, 300, 70), (12, 2, 2, 600, 230)])
def test_query_gradients_beside_larger_keys(ctx, r, d, B, H, Hkv, L, window):
    """Queries that see the first keys and their window, between them keys that only other queries of the same wavefront see: these
    are 2^r times as large, and the queries 2^-r times, so that all scores are ordinary ones."""
    sinks, at = 4, slice(96, 128)
    q, k, v, g = _inputs(np.random.default_rng(r + d + 400), B, H, Hkv, L, L, d)
    q *= np.float32(2.0 ** -r)
    k[:, :, at] *= np.float32(2.0 ** r)
    got = _forward_backward(ctx, q, k, v, g, _scale(d), window, sinks)
    k[:, :, at] = 0
    q, k, v, g = _ends(q, k, v, g)
    want = attention(q, k, v, _scale(d), window, sinks, dout=g)
    for rows in (slice(0, 96), slice(127 + window, L)):
        _compare(got, want, ["dq"], rows, "queries beside larger keys")


@pytest.mark.parametrize("r", SPREADS)
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("B,H,Hkv,L,window,length", [(40, 2, 2, 230, 4, 230), (40, 2, 2, 230, 4, 198), (14, 4, 1, 197, 3, 197), (9, 4, 2, 461, 10, 461)])
def test_last_rows_behind_larger_values(ctx, r, d, B, H, Hkv, L, window, length):
    """A tile that ends with fewer than 32 keys, 2^-r times as large as those of the tiles before it: its missing rows have no size."""
    q, k, v, g = _inputs(np.random.default_rng(r + d + 500), B, H, Hkv, L, L, d)
    last = length // 32 * 32
    v[:, :, last:] *= np.float32(2.0 ** -r)
    got = _forward_backward(ctx, q, k, v, g, _scale(d), window, lengths=[length] * B)
    v[:, :, :last] = 0
    q, k, v, g = _ends(q, k, v, g)
    want = attention(q, k, v, _scale(d), window, lengths=[length] * 2, dout=g)
    _compare(got, want, ("out", "dq"), slice(last + window - 1, L), "the last rows")
    # (a key's gradient takes in all queries that see it)
    _compare(got, want, ("dk", "dv"), slice(last + window - 1, L), "the last rows")
