"""The training operators' plain form in 64 bits, with a bound on what fp32
kernels may be off, element by element, from the arithmetic they do.

Products.  The tensor-core kernels take a product of two fp32 numbers as three
products of their fp16 halves (hi rounded to nearest, lo the rest rounded to
nearest): each operand is represented to 2^-22 of its value, so two cost
2^-21, and the dropped lo * lo is at most 2^-22.  (The weights' hi is
truncated, so theirs are represented to 2^-21; the chain below is counted long
enough for that: 12 accumulations follow one another per 64 columns, 24 in all
for 128, of which the weights' products take 12.)  A sum over head_dim or over
64 partners is a chain of at most 24 accumulations in fp32 that truncate, 2^-23
of the running sum of magnitudes each.  The row-wise kernels round d products
and sums in fp32, 2^-24 each.  So a dot product is off by at most

    EPS(d) * sum |a_c b_c|,   EPS(d) = max(2^-21 + 2^-22 + 24 * 2^-23, (d + 1) * 2^-24).

An operand 2^-39 below the largest of its 64 rows loses bits: an absolute
2^-40 of that largest value per element (SMALL), added to the magnitudes.

Scores.  x = scale * (q . k) + bias in powers of two: four more roundings, 2^-24
each, of the terms' magnitudes (the factor, the sum, the maximum, the
exponent's argument), so dx = EPS * A + 4 * 2^-24 * (A + |bias| + |m|) with
A = scale * sum |q_c k_c|.  The exponential (ex2.approx) is good to 2^-22, and
p = e^x / sum e^x has the relative error 2 * max dx + 2^-21 + (keys + 8) * 2^-24.
Everything behind p follows from p's error by the product rule.
"""
from __future__ import annotations

import math

import numpy as np

import raya_b200 as rb

U = 2.0 ** -24


def eps(d):
    return max(2.0 ** -21 + 2.0 ** -22 + 24 * 2.0 ** -23, (d + 1) * U)


def small(x):
    """2^-40 of the largest value of each (batch, head) slice, [b, h, 1, 1]."""
    return 2.0 ** -40 * np.abs(x).max(axis=(2, 3), keepdims=True) if x.size else np.zeros(x.shape[:2] + (1, 1))


def allowed(mask, block, seq, valid):
    i, j = np.arange(seq)[:, None], np.arange(seq)[None, :]
    if mask.kind == rb._lib.MASK_BLOCK:
        m = np.abs(i // block - j // block) <= mask.param
    elif mask.kind == rb._lib.MASK_WINDOW:
        m = np.abs(i - j) <= mask.param
    else:
        m = np.ones((seq, seq), bool)
    return m[None, None] & (i < valid[:, None, None, None]) & (j < valid[:, None, None, None])


def buckets_of(rel, buckets, max_distance):
    """bucket(rel) from the definition, in whole numbers."""
    half, first = buckets // 2, buckets // 4
    rest = half - first
    out = np.zeros(rel.shape, np.int64)
    for n in np.unique(np.abs(rel)):
        n = int(n)
        k = n
        if n >= first:  # the last k with n >= first (max / first)^(k / rest)
            k = first
            while k + 1 < half and n ** rest >= first ** (rest - (k + 1 - first)) * max_distance ** (k + 1 - first):
                k += 1
        out[np.abs(rel) == n] = k
    return out + (rel > 0) * half


def reference(mask, block, scale, valid, q, k, v, dout=None, table=None, max_distance=128):
    """{name: (value, bound)} in 64 bits for [b, h, s, d] arrays; valid is an int array [b]."""
    b, h, s, d = q.shape
    rows = np.arange(s)[None, None, :, None] < valid[:, None, None, None]
    q, k, v = (np.where(rows, x, 0).astype(np.float64) for x in (q, k, v))
    see = allowed(mask, block, s, valid)
    rel = np.arange(s)[None, :] - np.arange(s)[:, None]
    bias = np.zeros((h, s, s))
    if table is not None:
        ids = buckets_of(rel, table.shape[1], max_distance)
        t = np.where(table <= -(2.0 ** 100), -np.inf, table.astype(np.float64))
        bias = t[:, ids]
    see = np.broadcast_to(see & np.isfinite(bias)[None], (b, h, s, s))
    bias = np.where(np.isfinite(bias), bias, 0.0)[None]
    e = eps(d)
    x = np.where(see, scale * (q @ k.swapaxes(-1, -2)) + bias, -np.inf)
    m = x.max(-1, keepdims=True) if s else x.sum(-1, keepdims=True)
    m0 = np.where(np.isfinite(m), m, 0.0)
    w = np.exp(x - m0)
    l = w.sum(-1, keepdims=True)
    p = w / np.where(l > 0, l, 1)
    a = abs(scale) * ((np.abs(q) + small(q)) @ (np.abs(k) + small(k)).swapaxes(-1, -2))
    dx = np.where(see, e * a + 4 * U * (a + np.abs(bias) + np.abs(m0)), 0.0)
    dxm = dx.max(-1, keepdims=True) if s else dx.sum(-1, keepdims=True)
    n = see.sum(-1, keepdims=True)
    dp_rel = 2 * dxm + 2.0 ** -21 + (n + 8) * U
    out = p @ v
    va = np.abs(v) + small(v)
    got = {"out": (out, (dp_rel + e + (n + 8) * U) * (p @ va)), "m": (m, np.where(n > 0, dxm + 2 * U * np.abs(m0), 0)),
           "l": (l, l * dp_rel)}
    if dout is None:
        return got
    g = np.where(rows, dout, 0).astype(np.float64)
    ga = np.abs(g) + small(g)
    dp = g @ v.swapaxes(-1, -2)
    delta = (g * out).sum(-1, keepdims=True)
    da = ga @ va.swapaxes(-1, -2)
    # out enters delta as the caller gives it: rounded to fp32, and off by its own bound
    ddelta = (np.abs(g) * (got["out"][1] + (d + 2) * U * np.abs(out))).sum(-1, keepdims=True)
    ds = p * (dp - delta)
    # a weight far below its row's largest is held to 2^-24 of that one (fp16's smallest steps)
    pe = p * dp_rel + 2.0 ** -30 * p.max(-1, keepdims=True, initial=0) * see
    dse = p * (e * da + ddelta + 2 * U * (np.abs(dp) + np.abs(delta))) + pe * (np.abs(dp) + np.abs(delta))
    ta = dse + (e + (n.max(initial=0) + 8) * U) * np.abs(ds)
    # ds is held in fp16 halves to 2^-38 of the bound on it, |g_i| max |v_j| + |delta_i| with g = dout / l
    most = np.where(n > 0, (np.sqrt((g * g).sum(-1, keepdims=True)) * np.sqrt((v * v).sum(-1)).max(-1, initial=0)[..., None, None] + np.abs(delta))
                    / np.where(l > 0, l, 1), 0.0)
    lost = 2.0 ** -38
    taq, tak = ta + lost * most * see, ta + lost * most.max(-2, initial=0, keepdims=True) * see
    got["dq"] = (scale * (ds @ k), abs(scale) * (taq @ (np.abs(k) + small(k))))
    got["dk"] = (scale * (ds.swapaxes(-1, -2) @ q), abs(scale) * (tak.swapaxes(-1, -2) @ (np.abs(q) + small(q))))
    got["dv"] = (p.swapaxes(-1, -2) @ g, (pe + (e + (s + 8) * U) * p).swapaxes(-1, -2) @ ga)
    if table is not None:
        t, tb = np.zeros((2,) + table.shape)
        for c in range(table.shape[1]):
            hit = ids == c
            t[:, c] = ds[..., hit].sum((0, 2))
            # one rounding for each of a thread's at most `rows` values of a bucket, 64 of its block's
            tb[:, c] = (dse + (s + 64) * U * np.abs(ds))[..., hit].sum((0, 2))
        got["dtable"] = (t, tb)
    return got


def close(got, want, what):
    """got within the bound of want = (value, bound), plus one rounding of the result."""
    value, bound = want
    got = np.asarray(got, np.float64).reshape(value.shape)
    fine = np.isfinite(value)
    assert np.array_equal(got[~fine], value[~fine]), f"{what}: non-finite values differ"
    assert np.isfinite(got[fine]).all(), f"{what}: non-finite output"
    off = np.abs(got - np.where(fine, value, 0))[fine]
    most = (np.broadcast_to(bound, value.shape) + 2 * U * np.abs(np.where(fine, value, 0)))[fine] + 1e-37
    worst = float((off / most).max(initial=0))
    assert worst <= 1, f"{what}: {worst:.2f} times its bound (largest difference {off.max():.3e})"
    return worst


def scale_of(d):
    return 1.0 / math.sqrt(d)
