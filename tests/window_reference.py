"""Attention with a sliding window in 64 bits, with bounds on what fp32 arithmetic may be off by.

The bounds follow the arithmetic, worst case: a sum of n fp32 products is off by at most (n + c) u sum |a b| with
u = 2^-24 (c = 16 covers the scaling of q, the change to base 2, and products formed from split operands, whose dropped
parts are below 2^-24 of each product); an error e in the scores of a row changes its weights by at most a factor
exp(2 e), the exponential itself adds 4 u (1 + |s|); everything else is carried through the formulas in absolute values.

Operands are split into two fp16 planes under a power of two (x 2^a = h + l).  h takes 11 bits, l what is left, in steps of 2^-24
at the least: beside 2^-23 of x (in c above), a value is off by half such a step, 2^-25 2^-a.  What shares the power has a
largest value of at least 2^11 2^-a (rows read together: 2^-36 of the largest; 2^14 for a row alone, less).  Weights of the
forward pass are at most 2^15 and stand for 2^7 / (the largest so far) or more: each is off by at most 2^-32 of the row's sum.
Weights of dv are 2^13 w, or a power that puts the column's first largest at 2^8: off by 2^-38 or 2^-33 of the largest in the
column; dS, with such a power always, by 2^-33 of the largest in its row (dq) or column (dk).  These absolute errors, times
the other operand's absolute values, are added to the bounds: they matter where values that are summed differ in size."""
import numpy as np

U = 2.0 ** -24


def visible(Lq, Lk, window, sinks, q_offset, length):
    p = np.arange(Lq)[:, None] + q_offset
    j = np.arange(Lk)[None, :]
    return (j <= p) & ((j > p - window) | (j < sinks)) & (j < length)


def attention(q, k, v, rT, window, sinks=0, q_offset=0, lengths=None, dout=None):
    """q [B,H,Lq,d], k, v [B,Hkv,Lk,d] (fp32 or fp64).  Returns {name: (value, bound)} for out and, with dout, dq, dk, dv."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    B, H, Lq, d = q.shape
    Hkv, Lk = k.shape[1], k.shape[2]
    res = {"out": (np.zeros_like(q), np.zeros_like(q))}
    if dout is not None:
        dout = np.asarray(dout, np.float64)
        res.update(dq=(np.zeros_like(q), np.zeros_like(q)), dk=(np.zeros_like(k), np.zeros_like(k)),
                   dv=(np.zeros_like(k), np.zeros_like(k)))
    for b in range(B):
        length = Lk if lengths is None else max(0, min(int(lengths[b]), Lk))
        see = visible(Lq, Lk, window, sinks, q_offset, length)
        n = see.sum(1, keepdims=True)
        for h in range(H):
            kh, vh = np.where(np.arange(Lk)[:, None] < length, k[b, h * Hkv // H], 0), np.where(
                np.arange(Lk)[:, None] < length, v[b, h * Hkv // H], 0)
            s = q[b, h] @ kh.T * rT
            most = lambda x: np.abs(x).max(initial=0)
            plane = lambda x, y: 2.0 ** -36 * (most(x) * np.abs(y).sum(1)[None] + most(y) * np.abs(x).sum(1)[:, None])
            e_s = abs(rT) * ((d + 16) * U * (np.abs(q[b, h]) @ np.abs(kh).T) + plane(q[b, h], kh)) + 4 * U * (1 + np.abs(s))
            e_s = np.where(see, e_s, 0).max(1, keepdims=True, initial=0)
            w = np.exp(np.where(see, s, -np.inf) - np.where(see, s, -np.inf).max(1, keepdims=True, initial=-1e300))
            w /= np.where(n > 0, w.sum(1, keepdims=True), 1)
            e_w = np.expm1(2 * e_s) + (n + 16) * U                  # relative, of every weight of the row
            out = w @ vh
            e_out = (e_w + (n + 16) * U) * (w @ np.abs(vh)) + 2.0 ** -32 * (see @ np.abs(vh)) + 2.0 ** -36 * most(vh) * (n > 0)
            res["out"][0][b, h], res["out"][1][b, h] = out, e_out
            if dout is None:
                continue
            g = dout[b, h]
            dP, D = g @ vh.T, (g * out).sum(1, keepdims=True)
            e_D = (d + 16) * U * (np.abs(g) * (w @ np.abs(vh))).sum(1, keepdims=True) + (np.abs(g) * e_out).sum(1, keepdims=True)
            dS = w * (dP - D)
            e_dS = w * (e_w * np.abs(dP - D) + (d + 16) * U * (np.abs(g) @ np.abs(vh).T) + plane(g, vh) + e_D
                        + 4 * U * (np.abs(dP) + np.abs(D)))
            size, qh = np.abs(dS), q[b, h]
            top = lambda x, axis: x.max(axis, keepdims=True, initial=0)
            e_q = 2.0 ** -33 * top(size, 1) * (see @ np.abs(kh)) + 2.0 ** -36 * most(kh) * size.sum(1, keepdims=True)
            e_k = 2.0 ** -33 * top(size, 0).T * (see.T @ np.abs(qh)) + 2.0 ** -36 * most(qh) * size.sum(0)[:, None]
            e_v = np.maximum(2.0 ** -38, 2.0 ** -33 * top(w, 0).T) * (see.T @ np.abs(g)) + 2.0 ** -36 * most(g) * w.sum(0)[:, None]
            many = see.sum(0)[:, None] * (H // Hkv)                  # terms of a dk, dv element over the group
            res["dq"][0][b, h] = dS @ kh * rT
            res["dq"][1][b, h] = abs(rT) * ((e_dS + (n + 16) * U * np.abs(dS)) @ np.abs(kh) + e_q)
            hk = h * Hkv // H
            res["dk"][0][b, hk] += dS.T @ q[b, h] * rT
            res["dk"][1][b, hk] += abs(rT) * (e_dS.T @ np.abs(q[b, h]) + (many + 16) * U * (np.abs(dS).T @ np.abs(q[b, h])) + e_k)
            res["dv"][0][b, hk] += w.T @ g
            res["dv"][1][b, hk] += (w * e_w).T @ np.abs(g) + (many + 16) * U * (w.T @ np.abs(g)) + e_v
    return res


def assert_within(got, want, what):
    value, bound = want
    got = np.asarray(got, np.float64)
    assert got.shape == value.shape, (what, got.shape, value.shape)
    off = np.abs(got - value)
    bad = ~(off <= bound + 1e-37)
    if bad.any():
        i = np.unravel_index(int(np.argmax(np.where(np.isnan(off), np.inf, off - bound))), off.shape)
        raise AssertionError("%s: %d of %d outside; at %s got %.9g, want %.9g +- %.2g" % (
            what, bad.sum(), bad.size, i, got[i], value[i], bound[i]))
