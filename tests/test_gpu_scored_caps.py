"""Capped scores of every size against the 64-bit oracle, with a bound per key (needs an MI355X).

The bounds are asserted to lie far below the outputs: zeros, or uniform attention, fail.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from _scored import Pool, slopes_of
from engine.kernels.scored_attention import (paged_attention_decode_scored,
                                             paged_attention_prefill_scored)
from oracle.scored_attention_oracle import attend_bound

pytestmark = pytest.mark.gpu

CAPS = [1e-42, 1e-30, 1e-3, 0.5, 5.0, 50.0, 128.0, 128.0001, 200.0, 1e3, 1e4, 1e5, 1e6, 1e8, 1e12, 1e30, 1e38]


def near(got, want, bound):
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all()
    off = np.abs(got - want) - bound
    assert (off <= 0).all(), f"{off.max():.3e} over the bound at {np.unravel_index(off.argmax(), off.shape)}"
    assert np.median(bound) < 0.15 * np.median(np.abs(want))


def decode(pool, q, scale, softcap, slopes=None, window=0):
    out = paged_attention_decode_scored(q, pool.k, pool.v, pool.tables, pool.seq_lens, scale, softcap, slopes,
                                        window)
    host, s = q.cpu().numpy(), None if slopes is None else slopes.cpu().numpy()
    for b, n in enumerate(pool.lens):
        want, bound = attend_bound(host[b:b + 1], *pool.rows(b), [n - 1], [n - window if window else 0], [n], scale,
                                   float(np.float32(softcap)), s)
        near(out[b:b + 1], want, bound)
    return out


def prefill(pool, q, new, scale, softcap, slopes=None, window=0, ends=None, pick=None):
    loc = np.concatenate([[0], np.cumsum(new)])
    out = paged_attention_prefill_scored(q, pool.k, pool.v, pool.tables, pool.seq_lens, pool.ints(loc), max(new),
                                         scale, softcap, slopes, window, None,
                                         None if ends is None else pool.ints(ends))
    host, s = q.cpu().numpy(), None if slopes is None else slopes.cpu().numpy()
    for b in range(len(new)) if pick is None else pick:
        r = slice(loc[b], loc[b + 1])
        pos = np.arange(pool.lens[b] - new[b], pool.lens[b])
        first = np.maximum(pos - window + 1, 0) if window else np.zeros_like(pos)
        want, bound = attend_bound(host[r], *pool.rows(b), pos, first, pos + 1 if ends is None else ends[r], scale,
                                   float(np.float32(softcap)), s, scaled=False)
        near(out[r], want, bound)
    return out


@pytest.mark.parametrize("softcap", CAPS)
def test_decode_at_every_cap(cuda_device, softcap):
    for d, bs in ((64, 16), (128, 5)):
        pool = Pool([700, 3, 129, 2500], 2, d, bs, cuda_device, seed=d)
        pool.k[pool.table[0, 1], 2] = 0  # a product of 0
        q = pool.queries(4, 8, spread=4.0)
        out = decode(pool, q, d ** -0.5, softcap)
        if softcap >= 1e30:  # no cap at all
            plain = decode(pool, q, d ** -0.5, 0.0)
            assert torch.equal(out, plain)
        decode(pool, q, d ** -0.5, softcap, slopes_of(8, cuda_device), 100)


@pytest.mark.parametrize("softcap", CAPS)
def test_prefill_at_every_cap(cuda_device, softcap):
    pool = Pool([150, 70], 2, 64, 16, cuda_device)
    new = [60, 70]
    pool.k[pool.table[0, 1], 2] = 0  # a product of 0
    q = pool.queries(130, 8, spread=4.0)
    out = prefill(pool, q, new, 0.125, softcap)
    if softcap >= 1e30:
        assert torch.equal(out, prefill(pool, q, new, 0.125, 0.0))


@pytest.mark.parametrize("heads,hkv,d,bs", [(14, 2, 64, 16), (8, 2, 128, 16), (4, 2, 32, 16), (4, 2, 256, 5),
                                            (8, 2, 128, 8)])
def test_wide_caps_with_bias_windows_and_ends(cuda_device, heads, hkv, d, bs):
    """Few and many columns, keys split over workgroups, prefixes seen as a whole."""
    slopes = slopes_of(heads, cuda_device)
    for lens, new, pick in (([200, 90], [50, 90], None), ([160] * 12, [130] * 12, [0, 11]), ([2600], [9], None)):
        pool = Pool(lens, hkv, d, bs, cuda_device, seed=d)
        q = pool.queries(sum(new), heads, spread=4.0)
        ends = np.concatenate([np.maximum(np.arange(n - k, n) + 1, n - 7) for n, k in zip(lens, new)])
        for f in (dict(softcap=300.0), dict(softcap=2e5, slopes=slopes), dict(softcap=1e4, window=40),
                  dict(softcap=3e6, slopes=slopes, ends=ends)):
            prefill(pool, q, new, d ** -0.5, pick=pick, **f)


def test_large_capped_scores(cuda_device):
    """Scores of thousands, with caps far below, near and far above them."""
    pool = Pool([700, 30], 2, 128, 16, cuda_device)
    q = pool.queries(2, 8, spread=300.0)
    for softcap in (0.5, 50.0, 3000.0, 1e6):
        decode(pool, q, 1.0, softcap)
    new = [20, 30]
    q = pool.queries(50, 8, spread=300.0)
    for softcap in (0.5, 50.0, 3000.0, 1e6):
        prefill(pool, q, new, 1.0, softcap)


@pytest.mark.parametrize("scale", [2.0 ** -130, 1e-30, 1e30, 2.0 ** 127])
def test_far_scales(cuda_device, scale):
    """Scores around 1 of tiny and huge scales, capped and not: finite, and as at scale 1."""
    pool = Pool([300, 40], 2, 64, 16, cuda_device)
    q = pool.queries(2, 8, spread=4.0)
    small = scale < 1
    for softcap in (0.0, 2.0 * scale if small else 50.0, 1e3):
        out = paged_attention_decode_scored(q, pool.k, pool.v, pool.tables, pool.seq_lens, scale, softcap)
        more = paged_attention_prefill_scored(q, pool.k, pool.v, pool.tables, pool.seq_lens, pool.ints([0, 1, 2]), 1,
                                              scale, softcap)
        if small:  # every key weighs the same
            for b in range(2):
                v = pool.rows(b)[1].mean(axis=0).repeat(4, axis=0)
                for x in (out, more):
                    assert (np.abs(x[b].double().cpu().numpy() - v) <= np.abs(v) * 2.0 ** -11 + 2e-3).all()
        elif softcap:  # keys of positive products weigh the same, the others nothing
            assert torch.isfinite(out).all() and torch.isfinite(more).all()
            assert (out.float() - more.float()).abs().max() < 4e-3
