"""Scores of any size that fp32 holds, without a cap (needs an MI355X)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from _scored import Pool
from engine.kernels.scored_attention import paged_attention_decode_scored

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
