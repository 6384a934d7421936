"""Attention of several new tokens per sequence over the 8-bit pool, and a drafted decode step
over it from end to end, against the 64-bit oracle (needs an MI355X).

Tolerances are the oracle's own bound per element (oracle/fp8_cache_oracle.py, attention).
Probabilities here keep all of fp16's bits down to 2^-22 of a running maximum that may lie up
to 2^8 under the true one, so each below is off by at most 2^-33 of the largest (half of fp16's
smallest step, 2^-25, over 2^8): below the bound's (L / 32 + 64) 2^-24 for every length.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from _fp8_pool import Fp8Pool, int32, starts_of
from engine.kernels import _native
from engine.kernels.paged_attention import paged_attention_prefill
from engine.kernels.quantized_cache import (
    paged_attention_decode_fp8,
    paged_attention_prefill_fp8,
    paged_kv_write_fp8,
)
from engine.kernels.speculative import verify_drafts
from oracle import fp8_cache_oracle as oracle
from oracle.speculative_oracle import verify

pytestmark = pytest.mark.gpu


def queries(n, hq, d, seed, device):
    return torch.randn(n, hq, d, generator=torch.Generator().manual_seed(seed)).half().to(device)


def run(pool, q, new, scale):
    return paged_attention_prefill_fp8(q, *pool.args(), int32(starts_of(new), pool.device), max(new),
                                       scale)


def check(pool, q, new, scale, out=None):
    if out is None:
        out = run(pool, q, new, scale)
    want, tol = oracle.attention(pool.state(), q.double().cpu().numpy(), pool.tables, pool.lens,
                                 starts_of(new), pool.bs, scale, bound=True)
    got = out.double().cpu().numpy()
    assert np.isfinite(got).all()
    off = np.abs(got - want)
    assert (off <= tol).all(), f"{(off / np.maximum(tol, 1e-30)).max():.3g} of the bound"
    return out


SHAPES = [(14, 2, 64, 16), (28, 4, 128, 16), (8, 8, 128, 16), (32, 2, 32, 16), (16, 2, 256, 16),
          (14, 2, 64, 8), (14, 2, 64, 32), (6, 2, 64, 5), (3, 1, 64, 48), (6, 3, 64, 1), (4, 4, 32, 32)]


@pytest.mark.parametrize("hq,hkv,d,bs", SHAPES)
def test_matches_oracle(cuda_device, hq, hkv, d, bs):
    """Prefix and suffix, whole prompts, single tokens, no new tokens, in one launch."""
    lens, new = [100, 17, 400, 64, 33, 150, 1, 0], [36, 17, 70, 1, 0, 150, 1, 0]
    pool = Fp8Pool(lens, hkv, d, bs, seed=hq + d + bs, device=cuda_device)
    check(pool, queries(sum(new), hq, d, 1, cuda_device), new, d ** -0.5)


@pytest.mark.parametrize("hq,hkv,d,bs", SHAPES)
def test_drafts(cuda_device, hq, hkv, d, bs):
    """A few tokens each at the end of contexts of all lengths."""
    lens = [5, 6, 16, 17, 33, 130, 257, 900, 2100]
    new = [5, 5, 1, 4, 5, 2, 8, 5, 3]
    pool = Fp8Pool(lens, hkv, d, bs, seed=hq + d, device=cuda_device)
    check(pool, queries(sum(new), hq, d, 2, cuda_device), new, d ** -0.5)


@pytest.mark.parametrize("longest", [60, 2540])
@pytest.mark.parametrize("most", [1, 3, 9])
@pytest.mark.parametrize("seqs", [20, 40, 140, 290])
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (4, 2, 32), (6, 3, 128)])
def test_drafts_of_many_sequences(cuda_device, hq, hkv, d, seqs, most, longest):
    """One token each at most, and more, for pair counts around the compute units', tables of
    whole pairs and of ranges."""
    g = torch.Generator().manual_seed(seqs + most)
    new = torch.randint(0, most + 1, (seqs,), generator=g).tolist()
    new[seqs // 2] = most
    lens = [n + int(x) for n, x in zip(new, torch.randint(0, 50, (seqs,), generator=g))]
    lens[1], new[1] = longest, 1
    pool = Fp8Pool(lens, hkv, d, 16, seed=seqs, device=cuda_device)
    check(pool, queries(sum(new), hq, d, 3, cuda_device), new, d ** -0.5)


def test_split_keys(cuda_device):
    """One long context: its keys are split over workgroups; the same bits every time."""
    pool = Fp8Pool([9000], 2, 64, 16, seed=3, device=cuda_device)
    q = queries(6, 14, 64, 4, cuda_device)
    out = check(pool, q, [6], 0.125)
    for _ in range(3):
        assert torch.equal(run(pool, q, [6], 0.125), out)


def test_more_parts_than_a_merge_takes_at_once(cuda_device):
    pool = Fp8Pool([90000], 1, 32, 16, seed=4, device=cuda_device)
    q = queries(4, 16, 32, 5, cuda_device)
    out = check(pool, q, [4], 0.2)
    for _ in range(3):
        assert torch.equal(run(pool, q, [4], 0.2), out)


@pytest.mark.parametrize("scale", [4.0, 1e-3])
def test_peaked_and_flat(cuda_device, scale):
    pool = Fp8Pool([500, 40], 2, 64, 16, seed=5, device=cuda_device)
    check(pool, queries(100, 14, 64, 6, cuda_device), [70, 30], scale)


def test_cache_scales_of_the_whole_range(cuda_device):
    pool = Fp8Pool([700, 333], 2, 64, 16, seed=7, device=cuda_device)
    g = torch.Generator().manual_seed(1)
    pool.dvs.copy_(torch.exp2(torch.randint(-15, 8, pool.v_scale.shape, generator=g).float()))
    pool.dks.copy_(torch.exp2(torch.randint(-15, -6, pool.k_scale.shape, generator=g).float()))
    check(pool, queries(41, 14, 64, 8, cuda_device), [8, 33], 0.125)


def test_nan_in_rows_that_are_not_seen(cuda_device):
    """Behind the end, and in later tokens of the same sequence: only the rows that see a NaN
    become NaN."""
    lens, new = [60, 130, 20], [40, 9, 20]
    pool = Fp8Pool(lens, 2, 64, 16, seed=9, device=cuda_device)
    q = queries(sum(new), 14, 64, 10, cuda_device)
    used = np.zeros((pool.blocks, 16), dtype=bool)
    for b, n in enumerate(lens):
        for p in range(n):
            used[pool.tables[b, p // 16], p % 16] = True
    base = check(pool, q, new, 0.125)
    hole = torch.from_numpy(~used).to(cuda_device)
    for cache in (pool.dk, pool.dv):
        cache.view(torch.uint8)[hole] = 0xff
    unused = torch.from_numpy(~used.any(axis=1)).to(cuda_device)
    pool.dks[unused] = float("nan")
    pool.dvs[unused] = float("nan")
    assert torch.equal(run(pool, q, new, 0.125), base)
    # Sequence 0's token at position 50 (its row 30), and sequence 1's at 3 (seen by all rows).
    for cache, d in ((pool.dv, 5), (pool.dk, 63)):
        cache.view(torch.uint8)[pool.tables[0, 3], 2, 1, d] = 0x7f
        out = run(pool, q, new, 0.125)
        assert torch.equal(out[:, :7], base[:, :7]) and torch.equal(out[:30], base[:30])
        assert out[30:40, 7:].isnan().any(dim=2).all()
        assert torch.equal(out[40:], base[40:])
        cache.view(torch.uint8)[pool.tables[0, 3], 2, 1, d] = 0
    pool.dv.view(torch.uint8)[pool.tables[1, 0], 3, 0, 9] = 0xff
    out = run(pool, q, new, 0.125)
    assert out[40:49, :7].isnan().any(dim=2).all() and torch.equal(out[49:], base[49:])


def test_tables_lengths_and_rows_out_of_range(cuda_device):
    """Contexts shorter than their new rows (zeros), bad block ids (clamped), rows of no sequence
    (left alone)."""
    pool = Fp8Pool([64, 64, 30], 2, 64, 16, seed=11, device=cuda_device)
    pool.tables[0, 1] = -7
    pool.tables[1, 2] = pool.blocks + 5
    pool.dt = torch.from_numpy(pool.tables).to(cuda_device)
    pool.lens = [64, 5000, 3]
    pool.dl = int32(pool.lens, cuda_device)
    new = [10, 64, 8]
    q = queries(82, 14, 64, 12, cuda_device)
    out = check(pool, q, new, 0.125)
    assert not out[74:79].any() and out[79:].any()


def test_agrees_with_the_fp16_pool_and_with_decode(cuda_device):
    lens, new = [1, 100, 1000, 3000], [1, 1, 1, 1]
    pool = Fp8Pool(lens, 2, 64, 16, seed=13, device=cuda_device)
    q = queries(4, 14, 64, 14, cuda_device)
    out = check(pool, q, new, 0.125)
    dec = paged_attention_decode_fp8(q, *pool.args(), 0.125)
    check(pool, q, new, 0.125, out=dec)
    k = (pool.dk.float() * pool.dks[:, None, :, None]).half()
    v = (pool.dv.float() * pool.dvs[:, None, :, None]).half()
    ref = paged_attention_prefill(q, k, v, pool.dt, pool.dl, int32(starts_of(new), cuda_device), 1, 0.125)
    assert (out.float() - ref.float()).abs().max() <= 2e-2


@torch.inference_mode()  # as every capture among these tests: torch's generator state may be one of it
def test_strides_and_graph(cuda_device):
    lens, new = [90, 5000], [30, 7]
    pool = Fp8Pool(lens, 2, 64, 16, seed=15, device=cuda_device)
    q = queries(37, 14, 64, 16, cuda_device)
    base = check(pool, q, new, 0.125)
    wide = torch.zeros(37, 14, 3, 64, dtype=torch.float16, device=cuda_device)
    wide[:, :, 1] = q
    pool.dv = pool.dv.view(torch.uint8).transpose(1, 2).contiguous().view(pool.dv.dtype).transpose(1, 2)
    pool.dks = pool.dks.t().contiguous().t()
    assert torch.equal(run(pool, wide[:, :, 1], new, 0.125), base)
    starts = int32(starts_of(new), cuda_device)
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for part in (q, wide[:, :, 1]):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(paged_attention_prefill_fp8(part, *pool.args(), starts, 30, 0.125))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(4):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = run(pool, q, new, 0.125)
        torch.cuda.synchronize()
        for out in (*outs, eager):
            assert torch.equal(out, base)


def test_refusals(cuda_device):
    pool = Fp8Pool([20, 30], 2, 64, 16, seed=17, device=cuda_device)
    q = queries(5, 14, 64, 18, cuda_device)
    k, v, ks, vs, t, n = pool.args()
    starts = int32([0, 2, 5], cuda_device)
    for bad in ((q.float(), k, v, ks, vs, t, n, starts, 3), (q[:, :13], k, v, ks, vs, t, n, starts, 3),
                (q, k.view(torch.uint8), v, ks, vs, t, n, starts, 3),
                (q, k, v, ks[:, :1], vs, t, n, starts, 3), (q, k, v, ks, vs, t, n, starts[:2], 3),
                (q, k, v, ks, vs, t, n, starts.long(), 3), (q, k, v, ks, vs, t, n, starts, -1)):
        with pytest.raises(AssertionError):
            paged_attention_prefill_fp8(*bad, 0.125)
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(_native.NativeLibraryError, match="scale"):
            paged_attention_prefill_fp8(q, k, v, ks, vs, t, n, starts, 3, scale)
    assert paged_attention_prefill_fp8(q[:0], k, v, ks, vs, t, n, starts * 0, 0, 0.125).shape == (0, 14, 64)


def test_a_drafted_decode_step(cuda_device):
    """Write the drafts' rows, attend over the pool, verify, take the rejected tokens back, write
    and attend again: as a serving loop does, over three steps."""
    hq, hkv, d, bs, vocab, k = 8, 2, 64, 16, 512, 4
    lens0 = [37, 5, 140, 16]
    n = len(lens0)
    pool = Fp8Pool([m + 40 for m in lens0], hkv, d, bs, seed=19, device=cuda_device)
    want = pool.oracle()
    g = torch.Generator().manual_seed(20)
    head = torch.randn(hq * d, vocab, generator=g).to(cuda_device)
    lens = list(lens0)
    for step in range(3):
        # Rows of the last emitted token and k drafts of each sequence.
        new = [k + 1] * n
        now = [m + k + 1 for m in lens]
        rows = [torch.randn(n * (k + 1), hkv, d, generator=g).half().to(cuda_device) for _ in range(2)]
        q = torch.randn(n * (k + 1), hq, d, generator=g).half().to(cuda_device)
        args = (*pool.args()[:5], int32(now, cuda_device))
        starts = int32(starts_of(new), cuda_device)
        paged_kv_write_fp8(*rows, *args, starts)
        oracle.write(want, *(r.double().cpu().numpy() for r in rows), pool.tables, now,
                     starts_of(new), bs)
        out = paged_attention_prefill_fp8(q, *args, starts, k + 1, d ** -0.5)
        exact, tol = oracle.attention(want, q.double().cpu().numpy(), pool.tables, now,
                                      starts_of(new), bs, d ** -0.5, bound=True)
        assert (np.abs(out.double().cpu().numpy() - exact) <= tol).all()
        p = torch.softmax(out.float().view(n, k + 1, hq * d) @ head, dim=-1)
        draft = torch.softmax(torch.randn(n, k, vocab, generator=g) * 0.1, dim=-1).to(cuda_device)
        ids = p[:, :k].argmax(dim=-1)
        u, u_next = torch.rand(n, k, generator=g).to(cuda_device), torch.rand(n, generator=g).to(cuda_device)
        tokens, accepted = verify_drafts(p, draft, ids, u, u_next)
        wanted = verify(*(x.cpu().numpy() for x in (p, draft, ids, u, u_next)))
        assert np.array_equal(tokens.cpu().numpy(), wanted[0])
        assert np.array_equal(accepted.cpu().numpy(), wanted[1])
        lens = [m + 1 + int(a) for m, a in zip(lens, accepted.tolist())]
    got = pool.state()
    for name in want:
        assert np.array_equal(got[name], want[name])
