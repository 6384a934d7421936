"""Scores of any size that fp32 holds, without a cap (needs an MI355X)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from _scored import Pool
from engine.kernels.scored_attention import (paged_attention_decode_scored,
                                             paged_attention_prefill_scored)

pytestmark = pytest.mark.gpu

SIZES = range(10, 100, 3)  # scores of 2^10 and more in the exp2 domain


def made(device, d, lens, heads=8):
    """Queries and keys of equal elements."""
    pool = Pool(lens, 2, d, 16, device, seed=d)
    pool.k.fill_(1.0)
    return pool, ones(len(lens), heads, d, device)


def ones(rows, heads, d, device):
    """A little more from head to head: products that a scale makes inexact in either direction."""
    q = torch.linspace(1.0, 1.43, heads, device=device).half()
    return q[None, :, None].expand(rows, heads, d).contiguous()


@pytest.mark.parametrize("d", [64, 128])
def test_decode_of_equal_keys(cuda_device, d):
    """Their mean, whatever their score; one that is larger alone."""
    lens = [300, 33, 2500]
    pool, q = made(cuda_device, d, lens)
    means = [pool.rows(b)[1].mean(axis=0).repeat(4, axis=0) for b in range(3)]
    sizes = [np.abs(pool.rows(b)[1]).mean(axis=0).repeat(4, axis=0) for b in range(3)]
    for e in SIZES:
        scale = 1.37 * 2.0 ** e / (d * 1.4426950408889634)
        out = paged_attention_decode_scored(q, pool.k, pool.v, pool.tables, pool.seq_lens, scale)
        for b in range(3):  # fp32 sums of up to 2500 equal shares, rounded once
            off = np.abs(out[b].double().cpu().numpy() - means[b])
            assert (off <= np.abs(means[b]) * 2.0 ** -11 + sizes[b] * 2.0 ** -13 + 2.0 ** -24).all(), (e, b)
    for b, key in enumerate((17, 0, 1999)):
        pool.k[pool.table[b, key // 16], key % 16] = 2.0
    for e in SIZES:
        scale = 1.37 * 2.0 ** e / (d * 1.4426950408889634)
        out = paged_attention_decode_scored(q, pool.k, pool.v, pool.tables, pool.seq_lens, scale)
        for b, key in enumerate((17, 0, 1999)):
            assert torch.equal(out[b], pool.v[pool.table[b, key // 16], key % 16].repeat_interleave(4, dim=0)), (e, b)


@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("softcap", [0.0, 1e9])
def test_prefill_of_equal_keys(cuda_device, d, softcap):
    """Within the keys' values (fp32 holds such scores to some units only); one that is larger alone."""
    lens, new = [700, 200, 2300], [40, 200, 1]
    pool, _ = made(cuda_device, d, lens)
    q = ones(241, 8, d, cuda_device)
    loc = pool.ints([0, 40, 240, 241])
    rows = [pool.rows(b)[1] for b in range(3)]

    def run(e):
        scale = 1.37 * 2.0 ** e / (d * 1.4426950408889634)
        return paged_attention_prefill_scored(q, pool.k, pool.v, pool.tables, pool.seq_lens, loc, 200, scale, softcap)

    sizes = [e for e in SIZES if softcap == 0.0 or e < 25]
    for e in sizes:
        out = run(e).double().cpu().numpy()
        at = 0
        for b in range(3):
            for i in range(new[b]):
                v = rows[b][:lens[b] - new[b] + i + 1]
                lo, hi = (x.repeat(4, axis=0) for x in (v.min(axis=0), v.max(axis=0)))
                slack = 2.0 ** -10 * np.maximum(np.abs(lo), np.abs(hi))
                assert (out[at] >= lo - slack).all() and (out[at] <= hi + slack).all(), (e, b, i)
                if e < 11:  # scores within 2^-13: the mean to 2^-12
                    mean, size = v.mean(axis=0).repeat(4, axis=0), np.abs(v).mean(axis=0).repeat(4, axis=0)
                    assert (np.abs(out[at] - mean) <= np.abs(mean) * 2.0 ** -11 + size * 2.0 ** -11).all(), (b, i)
                at += 1
    keys = (17, 0, 1999)
    for b, key in enumerate(keys):
        pool.k[pool.table[b, key // 16], key % 16] = 2.0
    for e in sizes:
        out = run(e)
        for b, (r, key) in enumerate(zip((slice(0, 40), slice(40, 240), slice(240, 241)), keys)):
            v = pool.v[pool.table[b, key // 16], key % 16].repeat_interleave(4, dim=0)
            assert (out[r] == v).all(), (e, b)
