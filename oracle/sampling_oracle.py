"""Sampling from logits, in 64-bit numpy on the CPU (test infrastructure only).

Row by row from the definition: weights exp((z - max z) / T); entries ordered by logit,
largest first, equal ones by index; the first top_k; of them the shortest beginning that
weighs top_p of their sum; of those the ones with a weight of min_p and more. The token is
the first index whose cumulative kept weight exceeds u times the sum.
"""
from __future__ import annotations

import numpy as np


def kept_weights(z, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Weights of one row's entries, 0 where an entry is not kept."""
    z = np.where(np.isnan(z), -np.inf, np.asarray(z, dtype=np.float64))
    out = np.zeros(len(z))
    top = z.max()
    if top == -np.inf:
        return out
    if not temperature > 0:
        out[int(np.argmax(z))] = 1.0
        return out
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(z == top, 1.0, np.exp((z - top) / temperature))
    w = np.where(np.isnan(w) | (z == -np.inf), 0.0, w)
    order = np.lexsort((np.arange(len(z)), -z))
    order = order[z[order] > -np.inf]
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        sums = np.cumsum(w[order])
        order = order[:max(1, int(np.searchsorted(sums, top_p * sums[-1], side="left")) + 1)]
    if min_p > 0:
        order = order[w[order] >= min(min_p, 1.0)]
    out[order] = w[order]
    return out


def probabilities(z, **settings):
    w = kept_weights(z, **settings)
    return w / w.sum() if w.sum() > 0 else w


def sample(z, u, **settings):
    """(token, distance of u * sum from the next border over the sum).

    Weights below 2^-45 of the largest count as none.
    """
    w = kept_weights(z, **settings)
    w = np.where(w < 2.0 ** -45, 0.0, w)
    live = np.flatnonzero(w)
    if len(live) == 0:
        return 0, 1.0
    sums = np.cumsum(w[live])
    aim = float(u) * sums[-1]
    above = np.flatnonzero(sums > aim)  # (none for NaN)
    token = live[above[0]] if len(above) else live[-1]
    return int(token), float(np.abs(sums[:-1] - aim).min() / sums[-1]) if len(live) > 1 else 1.0
