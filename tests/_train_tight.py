"""Tighter bounds than tests/_train.py's for the gradients: what the kernels
may be off where weights are small, element by element.

As there, a dot product is off by EPS(d) of its terms' magnitudes, and an
operand absolutely by 2^-40 of the largest value of its own 64 rows (here of
those, not of the slice).  The weights p = w / l, w = e^(x - m):

    rel_ij = dx_ij + sum_j p_ij dx_ij + 2^-21 + (keys + 8) * 2^-24

since w is off by its own score's error and the exponential's 2^-22, and l by
its terms'; nothing in it is absolute, so a weight of 2^-60 is as good as one
of 1.

What meets the second operand on the tensor cores is held in two fp16 numbers,
to 2^-21 of itself (counted in EPS), or after scaling to 2^-24 (half a step of
hi and of lo).  For dk that is at most 2^-22 of the largest |ds| that the key
has.  For dv it is 2^-22 of the largest w that the key has had, each one in the
scale of its 64 queries' dout / l, whose exponents are known to a factor of 2:
2^-21 of w_s G_s / G with G the largest dout / l of 64 queries; queries without
a dout do not count.  ds of dq is
scaled by the bound |g_i| |v_j| + |delta_i| instead and held to 2^-37 of it: dq
sums over a row's keys, of which one has a weight of the row's size.  The
table's gradient takes ds in fp32.
"""
from __future__ import annotations

import numpy as np

from _train import U, allowed, buckets_of, eps, reference


def small(x):
    """2^-40 of the largest value of each element's 64 rows, [b, h, s, 1]."""
    return 2.0 ** -40 * spread(np.abs(x).max(-1, keepdims=True, initial=0), -2, np.max)


def magnitude(x):
    """|x| with what its representation may add to it; a zero is exact."""
    return np.where(x != 0, np.abs(x) + small(x), 0.0)


def spread(x, axis, join):
    """join over each 64 entries of an axis, repeated for each of them."""
    n = x.shape[axis]
    parts = [join(np.take(x, range(r, min(r + 64, n)), axis), axis=axis, keepdims=True) for r in range(0, n, 64)]
    return np.concatenate([np.repeat(p, min(64, n - 64 * i), axis) for i, p in enumerate(parts)], axis) if n else x


def tiles(x, axis):
    """The sum over each 64 entries of an axis, one entry for each."""
    return np.add.reduceat(x, range(0, x.shape[axis], 64), axis=axis)


def tops(x, axis):
    return np.maximum.reduceat(x, range(0, x.shape[axis], 64), axis=axis)


def tight(mask, block, scale, valid, q, k, v, dout, table=None, max_distance=128):
    """{name: (value, bound)}: the values of reference(), for dq, dk, dv and dtable with the bounds above."""
    full = reference(mask, block, scale, valid, q, k, v, dout, table, max_distance)
    b, h, s, d = q.shape
    rows = np.arange(s)[None, None, :, None] < valid[:, None, None, None]
    q, k, v, g = (np.where(rows, x, 0).astype(np.float64) for x in (q, k, v, dout))
    rel = np.arange(s)[None, :] - np.arange(s)[:, None]
    see, bias = allowed(mask, block, s, valid), np.zeros((h, s, s))
    if table is not None:
        ids = buckets_of(rel, table.shape[1], max_distance)
        bias = np.where(table <= -(2.0 ** 100), -np.inf, table.astype(np.float64))[:, ids]
    see = np.broadcast_to(see & np.isfinite(bias)[None], (b, h, s, s))
    bias = np.where(np.isfinite(bias), bias, 0.0)[None]
    e = eps(d)
    x = np.where(see, scale * (q @ k.swapaxes(-1, -2)) + bias, -np.inf)
    m = x.max(-1, keepdims=True)
    m0 = np.where(np.isfinite(m), m, 0.0)
    w = np.exp(x - m0)
    l = w.sum(-1, keepdims=True)
    some = np.where(l > 0, l, 1)
    p, n = w / some, see.sum(-1, keepdims=True)
    a = abs(scale) * (magnitude(q) @ magnitude(k).swapaxes(-1, -2))
    dx = np.where(see, e * a + 4 * U * (a + np.abs(bias) + np.abs(m0)), 0.0)
    # 1.01: the second order
    off = 1.01 * (dx + (p * dx).sum(-1, keepdims=True) + 2.0 ** -21 + (n + 8) * U)
    ga, va = some * magnitude(g / some), magnitude(v)
    dp, delta = g @ v.swapaxes(-1, -2), (g * full["out"][0]).sum(-1, keepdims=True)
    ddelta = (np.abs(g) * (full["out"][1] + (d + 2) * U * np.abs(full["out"][0]))).sum(-1, keepdims=True)
    ds = p * (dp - delta)
    dse = p * (e * (ga @ va.swapaxes(-1, -2)) + ddelta + 4 * U * (np.abs(dp) + np.abs(delta))) + p * off * np.abs(dp - delta)
    held = e + (s + 8) * U
    t = lambda y: y.swapaxes(-1, -2)  # noqa: E731
    gl = np.abs(g / some)
    most_g = tops(gl.max(-1, keepdims=True, initial=0), -2)  # [b, h, tiles, 1]
    live = np.abs(g).max(-1, keepdims=True, initial=0) > 0
    largest = (tops(w * (1 + off) * live, -2) * most_g).max(-2)[..., None]  # [b, h, keys, 1]
    lost = 2.0 ** -21 * largest * (tiles(gl, -2) / np.where(most_g > 0, most_g, 1)).sum(-2, keepdims=True)
    got = dict(full)
    got["dv"] = (full["dv"][0], t(p * (off + held)) @ ga + lost)
    dsm = (np.abs(ds) + dse).max(-2)[..., None]
    got["dk"] = (full["dk"][0], abs(scale) * (t(dse + held * np.abs(ds)) @ magnitude(q)
                                              + 2.0 ** -22 * dsm * np.abs(q).sum(-2, keepdims=True)))
    most = np.where(n > 0, (np.sqrt((g * g).sum(-1, keepdims=True)) * np.sqrt((v * v).sum(-1)).max(-1, initial=0)[..., None, None]
                            + np.abs(delta)) / some, 0.0)
    got["dq"] = (full["dq"][0], abs(scale) * ((dse + held * np.abs(ds) + 2.0 ** -37 * most * see) @ magnitude(k)))
    if table is not None:
        tb = np.zeros(table.shape)
        for c in range(table.shape[1]):
            tb[:, c] = (dse + (s + 64) * U * np.abs(ds))[..., ids == c].sum((0, 2))
        got["dtable"] = (full["dtable"][0], tb)
    return got
