"""Pools, queries and checks shared by the tests of the scored attention."""
from __future__ import annotations

import numpy as np
import torch

from engine.kernels.scored_attention import (paged_attention_decode_scored,
                                             paged_attention_prefill_scored)
from oracle.scored_attention_oracle import attend, context, tolerance


class Pool:
    """A paged fp16 pool with sequences of the given lengths in shuffled blocks."""

    def __init__(self, lens, hkv, d, bs, device, seed=0, spare=3, width=0):
        rng = np.random.default_rng(seed)
        need = [-(-max(n, 0) // bs) for n in lens]
        self.blocks = sum(need) + spare
        self.lens, self.hkv, self.d, self.bs, self.device = list(lens), hkv, d, bs, device
        ids = rng.permutation(self.blocks)
        self.table = np.zeros((len(lens), max(need + [1, width])), dtype=np.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = ids[at:at + n]
            at += n
        g = torch.Generator(device=device).manual_seed(seed)
        shape = (self.blocks, bs, hkv, d)
        self.k = torch.randn(shape, generator=g, device=device, dtype=torch.float16)
        self.v = torch.randn(shape, generator=g, device=device, dtype=torch.float16)
        self.tables = torch.from_numpy(self.table).to(device)
        self.seq_lens = torch.tensor(self.lens, dtype=torch.int32, device=device)

    def queries(self, rows, heads, seed=1, spread=2.0):
        g = torch.Generator(device=self.device).manual_seed(seed)
        return spread * torch.randn(rows, heads, self.d, generator=g, device=self.device,
                                    dtype=torch.float16)

    def rows(self, b):
        """(k, v) of sequence b, float64."""
        n = min(max(self.lens[b], 0), self.table.shape[1] * self.bs)
        return [context(x.cpu().numpy(), self.table[b], n, self.bs) for x in (self.k, self.v)]

    def ints(self, values):
        return torch.tensor(np.asarray(values), dtype=torch.int32, device=self.device)


def slopes_of(heads, device):
    return torch.exp2(-8.0 / heads * torch.arange(1, heads + 1, device=device, dtype=torch.float32))


def near(got, want, spread, dim, softcap, scaled):
    got = got.double().cpu().numpy()
    off = np.abs(got - want) - tolerance(want, spread, dim, softcap, scaled)
    assert np.isfinite(got).all()
    assert (off <= 0).all(), f"{off.max():.3e} over the tolerance at {np.unravel_index(off.argmax(), off.shape)}"


def check_decode(pool, q, scale, softcap=0.0, slopes=None, window=0, starts=None, pick=None):
    """Against the oracle; the result."""
    out = paged_attention_decode_scored(
        q, pool.k, pool.v, pool.tables, pool.seq_lens, scale, softcap, slopes, window,
        None if starts is None else pool.ints(starts))
    host_q = q.cpu().numpy()
    host_slopes = None if slopes is None else slopes.cpu().numpy()
    for b in range(len(pool.lens)) if pick is None else pick:
        kk, vv = pool.rows(b)
        n = len(kk)
        first = 0 if starts is None else starts[b]
        if window:
            first = max(first, n - window)
        want, spread = attend(host_q[b:b + 1], kk, vv, [n - 1], [first], [n], scale, softcap, host_slopes)
        near(out[b:b + 1], want, spread, pool.d, softcap, True)
    return out


def check_prefill(pool, q, new, scale, softcap=0.0, slopes=None, window=0, starts=None, ends=None,
                  pick=None):
    """Against the oracle; the result. starts, ends: numpy per row, or None."""
    loc = np.concatenate([[0], np.cumsum(new)])
    out = paged_attention_prefill_scored(
        q, pool.k, pool.v, pool.tables, pool.seq_lens, pool.ints(loc), max(new), scale, softcap, slopes, window,
        None if starts is None else pool.ints(starts), None if ends is None else pool.ints(ends))
    host_q = q.cpu().numpy()
    host_slopes = None if slopes is None else slopes.cpu().numpy()
    for b in range(len(pool.lens)) if pick is None else pick:
        kk, vv = pool.rows(b)
        r = slice(loc[b], loc[b + 1])
        pos = np.arange(len(kk) - new[b], len(kk))
        first = np.zeros(new[b], dtype=np.int64) if starts is None else np.asarray(starts)[r]
        end = pos + 1 if ends is None else np.asarray(ends)[r]
        if window:
            first = np.maximum(first, pos - window + 1)
        want, spread = attend(host_q[r], kk, vv, pos, first, end, scale, softcap, host_slopes)
        near(out[r], want, spread, pool.d, softcap, False)
    return out
