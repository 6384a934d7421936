"""Verification of drafted tokens in 64 bits, sequence by sequence (test infrastructure only)."""
from __future__ import annotations

import numpy as np


def weights(p, q, certain=None):
    """max(p - q, 0) in float64, NaN as 0; with `certain` that index alone has no weight."""
    d = np.asarray(p, dtype=np.float64) - (0.0 if q is None else np.asarray(q, dtype=np.float64))
    w = np.where(d > 0, d, 0.0)
    if certain is not None and 0 <= certain < len(w):
        w[certain] = 0.0
    return w


def pick(w, u):
    """First index whose cumulative weight exceeds u * total, else the last with a weight, else 0."""
    c = np.cumsum(w)
    over = np.nonzero((c > np.float64(u) * c[-1]) & (w > 0))[0]
    some = np.nonzero(w > 0)[0]
    return int(over[0]) if len(over) else int(some[-1]) if len(some) else 0


def verify(target, draft, ids, accept_u, next_u, counts=None):
    """(tokens, accepted); arrays as verify_drafts takes them, as numpy fp32 / int64."""
    seqs, rows, vocab = target.shape
    k = rows - 1
    tokens = np.full((seqs, rows), -1, dtype=np.int64)
    accepted = np.zeros(seqs, dtype=np.int32)
    for b in range(seqs):
        d = k if counts is None else min(max(int(counts[b]), 0), k)
        n = 0
        while n < d:
            x = int(ids[b, n])
            if not 0 <= x < vocab:
                break
            q = 1.0 if draft is None else np.float64(draft[b, n, x])
            if not np.float64(accept_u[b, n]) * q < np.float64(target[b, n, x]):
                break
            n += 1
        if n < d:
            w = (weights(target[b, n], None, int(ids[b, n])) if draft is None
                 else weights(target[b, n], draft[b, n]))
            if not w.sum() > 0:
                w = weights(target[b, n], None)
        else:
            w = weights(target[b, n], None)
        tokens[b, :n] = ids[b, :n]
        tokens[b, n] = pick(w, next_u[b])
        accepted[b] = n
    return tokens, accepted
