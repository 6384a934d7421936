"""Attention with capped, biased and masked scores in 64 bits on the CPU (test infrastructure only).

Sequence by sequence and head by head, from the definition:
  s_j = cap(scale q.k_j) - slope |p - j|, cap(x) = softcap tanh(x / softcap),
  o = softmax(s) v over the keys of the row's interval; zeros where it holds none.
"""
from __future__ import annotations

import numpy as np


def context(cache, table, length, block_size):
    """The first `length` rows of a sequence, [length, kv heads, dim] float64."""
    ids = np.clip(table[:-(-length // block_size)], 0, cache.shape[0] - 1)
    return cache[ids].reshape(-1, *cache.shape[2:])[:length].astype(np.float64)


def attend(q, k, v, pos, first, end, scale, softcap=0.0, slopes=None):
    """(out [rows, heads, dim], bound on the spread of each) for rows at positions `pos`.

    The second is what rounding a probability or a score by one part of something may move:
    (sum_j p_j |v_j|, sum_i |q_i k_ij| scale at most, keys seen, largest |v| seen).
    """
    rows, heads, dim = q.shape
    g = heads // k.shape[1]
    out = np.zeros((rows, heads, dim))
    mass = np.zeros((rows, heads, dim))
    size = np.zeros((rows, heads))
    top = np.zeros((rows, heads))
    keys = np.zeros(rows, dtype=np.int64)
    for r in range(rows):
        lo, hi = max(0, int(first[r])), min(int(end[r]), len(k))
        if hi <= lo or pos[r] < 0:
            continue
        keys[r] = hi - lo
        j = np.arange(lo, hi)
        for h in range(heads):
            kk, vv = k[lo:hi, h // g], v[lo:hi, h // g]
            with np.errstate(invalid="ignore"):
                x = kk @ q[r, h].astype(np.float64) * scale
                size[r, h] = np.abs(kk * q[r, h].astype(np.float64)).sum(axis=1).max() * scale
                if softcap > 0:
                    x = softcap * np.tanh(x / softcap)
                if slopes is not None:
                    x = x - float(slopes[h]) * np.abs(pos[r] - j)
                p = np.exp(x - x.max())
                p /= p.sum()
                out[r, h] = p @ vv
                mass[r, h] = p @ np.abs(vv)
                top[r, h] = np.abs(vv).max()
    return out, (mass, size, keys, top)


def tolerance(out, spread, dim, softcap=0.0, scaled=True):
    """How far a result in fp16 may be off, element by element.

    The result's own rounding, 2^-11; probabilities rounded to fp16, half a step 2^-12, in
    numerator and denominator; scores in fp32, whose products' sums are off by dim 2^-24 of
    the sum of their sizes, and with a cap by a few 2^-24 of the cap. Probabilities that are
    not scaled up (`scaled` false) have steps of 2^-25 below 2^-14 of the largest.
    """
    mass, size, keys, top = spread
    score = (dim + 8) * 2.0 ** -24 * size + 8 * 2.0 ** -24 * softcap + 2.0 ** -20
    tol = np.abs(out) * 2.0 ** -11 + mass * (2.0 ** -11 + 2 * score[:, :, None]) + 2.0 ** -25
    if not scaled:
        tol = tol + (keys[:, None] * top)[:, :, None] * 2.0 ** -24
    return tol


def attend_bound(q, k, v, pos, first, end, scale, softcap=0.0, slopes=None, scaled=True):
    """(out, how far each element in fp16 may be off) as attend and tolerance, key by key.

    A score's products are off by dim 2^-24 of the sum of their sizes, of which a cap passes on
    its slope (the largest within that error); cap and bias add a few 2^-24 of what they give and,
    for caps up to 128, of the cap (2^-14 at most, an eighth of a probability's rounding). A
    probability is rounded to fp16, 2^-11 relative, and without being scaled up (`scaled` false) by
    2^-25 of the largest. Each moves the result by its share of p_j |v_j - out|.
    """
    rows, heads, dim = q.shape
    g = heads // k.shape[1]
    out = np.zeros((rows, heads, dim))
    bound = np.full((rows, heads, dim), 2.0 ** -25)
    step = 2.0 ** -24
    for r in range(rows):
        lo, hi = max(0, int(first[r])), min(int(end[r]), len(k))
        if hi <= lo or pos[r] < 0:
            continue
        away = np.abs(pos[r] - np.arange(lo, hi))
        for h in range(heads):
            kk, vv = k[lo:hi, h // g], v[lo:hi, h // g]
            each = kk * (q[r, h].astype(np.float64) * scale)
            x = each.sum(axis=1)
            off = (dim + 8) * step * np.abs(each).sum(axis=1)
            if softcap > 0:
                least = np.maximum(np.abs(x) - off, 0.0) / softcap
                off = off / np.cosh(np.minimum(least, 300.0)) ** 2
                x = softcap * np.tanh(x / softcap)
                off += 8 * step * (np.abs(x) + (softcap if softcap <= 128 else 0.0))
            if slopes is not None:
                bias = float(slopes[h]) * away
                x = x - bias
                off += 4 * step * (np.abs(bias) + np.abs(x))
            p = np.exp(x - x.max())
            off += 4 * step * np.abs(x - x.max()) + 2.0 ** -11
            flat = 0.0 if scaled else 2 * 2.0 ** -25 / p.sum()
            p /= p.sum()
            o = p @ vv
            out[r, h] = o
            # The shift itself and the sum's, at most all that there is.
            share = flat + np.minimum(p * np.expm1(np.minimum(2 * off, 700.0)), 1.0)
            bound[r, h] += np.abs(o) * 2.0 ** -11 + share @ np.abs(vv - o)
    return out, bound
