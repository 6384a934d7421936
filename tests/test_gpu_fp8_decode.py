"""Decode attention over the 8-bit pool against the 64-bit oracle (needs an MI355X).

Tolerances are the oracle's own bound per element (oracle/fp8_cache_oracle.py, attention):
fp32 sums, probabilities and outputs rounded to fp16.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from _fp8_pool import FP8, Fp8Pool, int32
from engine.kernels import _native
from engine.kernels.paged_attention import paged_attention_decode_batched
from engine.kernels.quantized_cache import paged_attention_decode_fp8
from oracle import fp8_cache_oracle as oracle

pytestmark = pytest.mark.gpu


def queries(n, hq, d, seed, device):
    return torch.randn(n, hq, d, generator=torch.Generator().manual_seed(seed)).half().to(device)


def check(pool, q, scale, out=None):
    if out is None:
        out = paged_attention_decode_fp8(q, *pool.args(), scale)
    want, tol = oracle.attention(pool.state(), q.double().cpu().numpy(), pool.tables, pool.lens,
                                 list(range(len(pool.lens) + 1)), pool.bs, scale, bound=True)
    got = out.double().cpu().numpy()
    assert np.isfinite(got).all()
    off = np.abs(got - want)
    assert (off <= tol).all(), f"{(off / tol).max():.3g} of the bound"
    return out


LENS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 255, 256, 257, 300, 700]


@pytest.mark.parametrize("hq,hkv,d,bs", [
    (14, 2, 64, 16), (28, 4, 128, 16), (8, 8, 128, 16), (32, 2, 32, 16), (16, 2, 256, 16),
    (14, 2, 64, 8), (14, 2, 64, 32), (6, 2, 64, 5), (3, 1, 64, 48), (6, 3, 64, 1), (4, 4, 128, 32),
    (16, 1, 256, 20), (7, 7, 32, 8)])
def test_matches_oracle(cuda_device, hq, hkv, d, bs):
    pool = Fp8Pool(LENS, hkv, d, bs, seed=hq + d + bs, device=cuda_device)
    check(pool, queries(len(LENS), hq, d, 1, cuda_device), d ** -0.5)


@pytest.mark.parametrize("hq,hkv,d,bs", [(14, 2, 64, 16), (4, 2, 32, 16), (8, 4, 64, 8), (5, 1, 128, 16)])
@pytest.mark.parametrize("n,longest", [(290, 211), (150, 211), (140, 1500), (40, 2300)])
def test_many_sequences(cuda_device, hq, hkv, d, bs, n, longest):
    """Pairs from less than half the compute units to more than all, short and long: enough that a
    workgroup takes two kv heads (head_dim 32 and 64), whole pairs and ranges."""
    lens = [(37 * i) % longest for i in range(n)]
    pool = Fp8Pool(lens, hkv, d, bs, seed=3, device=cuda_device, slack=1)
    check(pool, queries(len(lens), hq, d, 4, cuda_device), d ** -0.5)


@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (32, 2, 64), (64, 4, 32), (4, 2, 32), (8, 2, 128), (3, 1, 256)])
@pytest.mark.parametrize("n", [3, 90, 257, 700])
def test_ranges_of_mostly_empty_sequences(cuda_device, hq, hkv, d, n):
    """A long sequence among short and empty ones: range boundaries fall on what a pair costs
    beside its chunks, and the lengths are read in several turns."""
    g = torch.Generator().manual_seed(n)
    lens = torch.randint(0, 45, (n,), generator=g).tolist()
    lens[n // 3], lens[n - 1], lens[0] = 2700, 1333, 0
    pool = Fp8Pool(lens, hkv, d, 16, seed=n, device=cuda_device, slack=1)
    q = queries(n, hq, d, 5, cuda_device)
    out = check(pool, q, d ** -0.5)
    assert torch.equal(paged_attention_decode_fp8(q, *pool.args(), d ** -0.5), out)


@pytest.mark.parametrize("hq,hkv,d,bs,lens", [
    (14, 2, 64, 16, [24001]), (8, 1, 128, 16, [9000, 5, 0, 4097]), (16, 2, 256, 32, [5000, 260]),
    (2, 2, 64, 8, [3000, 2999, 1]), (4, 2, 32, 7, [2500]),
    (16, 1, 32, 16, [90000])])  # (the last: more parts of a pair than the merge takes at once)
def test_long_contexts_are_split(cuda_device, hq, hkv, d, bs, lens):
    pool = Fp8Pool(lens, hkv, d, bs, seed=5, device=cuda_device)
    q = queries(len(lens), hq, d, 6, cuda_device)
    out = check(pool, q, d ** -0.5)
    for _ in range(3):  # the same bits, whatever arrives last
        assert torch.equal(paged_attention_decode_fp8(q, *pool.args(), d ** -0.5), out)


@pytest.mark.parametrize("scale", [4.0, -0.125, 0.0, 1e-3])
def test_scales_of_the_softmax(cuda_device, scale):
    """Peaked, negative and flat: one token's weight, or everyone's."""
    pool = Fp8Pool([500, 40, 1], 2, 64, 16, seed=7, device=cuda_device)
    check(pool, queries(3, 14, 64, 8, cuda_device), scale)


def test_cache_scales_of_the_whole_range(cuda_device):
    """Neighbouring blocks whose scales lie orders of magnitude apart."""
    pool = Fp8Pool([900, 333], 2, 64, 16, seed=9, device=cuda_device)
    g = torch.Generator().manual_seed(1)
    pool.dvs.copy_(torch.exp2(torch.randint(-15, 8, pool.v_scale.shape, generator=g).float()))
    pool.dks.copy_(torch.exp2(torch.randint(-15, -6, pool.k_scale.shape, generator=g).float()))
    check(pool, queries(2, 14, 64, 10, cuda_device), 0.125)


def test_what_lies_behind_the_end_does_not_count(cuda_device):
    """NaN codes in the last block's free rows, in unused blocks and their scales."""
    lens = [5, 17, 300, 1, 0]
    pool = Fp8Pool(lens, 2, 64, 16, seed=11, device=cuda_device)
    q = queries(5, 14, 64, 12, cuda_device)
    used = np.zeros((pool.blocks, 16), dtype=bool)
    for b, n in enumerate(lens):
        for p in range(n):
            used[pool.tables[b, p // 16], p % 16] = True
    base = check(pool, q, 0.125)
    hole = torch.from_numpy(~used).to(cuda_device)
    for cache in (pool.dk, pool.dv):
        cache.view(torch.uint8)[hole] = 0x7f
    unused = torch.from_numpy(~used.any(axis=1)).to(cuda_device)
    pool.dks[unused] = float("nan")
    pool.dvs[unused] = float("inf")
    assert torch.equal(paged_attention_decode_fp8(q, *pool.args(), 0.125), base)


def test_a_nan_row_reaches_its_sequence_only(cuda_device):
    pool = Fp8Pool([40, 40], 2, 64, 16, seed=13, device=cuda_device)
    q = queries(2, 14, 64, 14, cuda_device)
    base = paged_attention_decode_fp8(q, *pool.args(), 0.125)
    pool.dk.view(torch.uint8)[pool.tables[0, 1], 3, 0] = 0x7f
    out = paged_attention_decode_fp8(q, *pool.args(), 0.125)
    assert out[0, :7].isnan().all() and torch.equal(out[0, 7:], base[0, 7:])
    assert torch.equal(out[1], base[1])


def test_tables_and_lengths_out_of_range(cuda_device):
    pool = Fp8Pool([64, 64, 30], 2, 64, 16, seed=15, device=cuda_device)
    pool.tables[0, 1] = -7
    pool.tables[1, 2] = pool.blocks + 5
    pool.dt = torch.from_numpy(pool.tables).to(cuda_device)
    pool.lens = [64, 5000, -3]
    pool.dl = int32(pool.lens, cuda_device)
    check(pool, queries(3, 14, 64, 16, cuda_device), 0.125)


def test_agrees_with_the_fp16_pool_of_the_same_values(cuda_device):
    lens = [1, 100, 1000, 3000]
    pool = Fp8Pool(lens, 2, 64, 16, seed=17, device=cuda_device)
    q = queries(4, 14, 64, 18, cuda_device)
    k = (pool.dk.float() * pool.dks[:, None, :, None]).half()
    v = (pool.dv.float() * pool.dvs[:, None, :, None]).half()
    ref = paged_attention_decode_batched(q, k, v, pool.dt, pool.dl, 0.125)
    out = check(pool, q, 0.125)
    check(pool, q, 0.125, out=ref)
    assert (out.float() - ref.float()).abs().max() <= 2e-2


def test_strides(cuda_device):
    """Query slices of a merged projection, one layer of a pool of several, transposed scales."""
    lens = [200, 33]
    pool = Fp8Pool(lens, 2, 64, 16, seed=19, device=cuda_device)
    q = queries(2, 14, 64, 20, cuda_device)
    base = check(pool, q, 0.125)
    wide = torch.zeros(2, 14, 3, 64, dtype=torch.float16, device=cuda_device)
    wide[:, :, 1] = q
    odd = torch.zeros(2, 14, 65, dtype=torch.float16, device=cuda_device)
    odd[..., 1:] = q
    layers = torch.zeros(pool.blocks, 3, 16, 2, 96, dtype=torch.uint8, device=cuda_device)
    layers[:, 1, :, :, 32:] = pool.dk.view(torch.uint8)
    k = layers.view(FP8)[:, 1, :, :, 32:]
    heads_first = pool.dv.view(torch.uint8).transpose(1, 2).contiguous().view(FP8).transpose(1, 2)
    scales = pool.dks.t().contiguous().t()
    table = torch.stack([pool.dt, pool.dt], dim=2)[..., 0]
    lens_ = torch.stack([pool.dl, pool.dl], dim=1)[:, 0]
    for qv in (wide[:, :, 1], odd[..., 1:]):
        out = paged_attention_decode_fp8(qv, k, heads_first, scales, pool.dvs, table, lens_, 0.125)
        assert torch.equal(out, base) and out.is_contiguous()


def test_offsets_past_32_bits(cuda_device):
    blocks, bs, hkv, d = 2 ** 16 + 9, 16, 32, 128  # 65,536 codes a block
    small = Fp8Pool([45], hkv, d, bs, seed=21, device=cuda_device)
    q = queries(1, 64, d, 22, cuda_device)
    base = paged_attention_decode_fp8(q, *small.args(), d ** -0.5)
    ids = [blocks - 1, 7, blocks - 3]
    big = []
    for cache in (small.dk, small.dv):
        x = torch.zeros(blocks, bs, hkv, d, dtype=torch.uint8, device=cuda_device)
        x[ids] = cache.view(torch.uint8)[small.tables[0].tolist()]
        big.append(x.view(FP8))
    for scale in (small.dks, small.dvs):
        x = torch.ones(blocks, hkv, device=cuda_device)
        x[ids] = scale[small.tables[0].tolist()]
        big.append(x)
    out = paged_attention_decode_fp8(q, *big, int32([ids], cuda_device), small.dl, d ** -0.5)
    assert torch.equal(out, base)


@torch.inference_mode()  # as every capture among these tests: torch's generator state may be one of it
def test_graphs_streams_and_eager_calls_share_nothing(cuda_device):
    """Two captured calls of other sizes replayed at once on two streams, eager calls beside them."""
    pools = [Fp8Pool([9000, 100], 2, 64, 16, seed=23, device=cuda_device),
             Fp8Pool([5000, 300, 7], 8, 128, 16, seed=24, device=cuda_device)]
    qs = [queries(2, 14, 64, 25, cuda_device), queries(3, 32, 128, 26, cuda_device)]
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for pool, q in zip(pools, qs):
        paged_attention_decode_fp8(q, *pool.args(), 0.1)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(paged_attention_decode_fp8(q, *pool.args(), 0.1))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for seed in range(4):
        for q in qs:
            q.copy_(queries(*q.shape, 30 + seed, cuda_device))
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = paged_attention_decode_fp8(qs[0], *pools[0].args(), 0.1)
        torch.cuda.synchronize()
        for pool, q, out in zip(pools, qs, outs):
            assert torch.equal(out, paged_attention_decode_fp8(q, *pool.args(), 0.1))
        assert torch.equal(eager, outs[0])
    check(pools[1], qs[1], 0.1, out=outs[1])
    for key, ws in _native._workspaces.items():
        if key[2] == _native.WS_DECODE_FP8:
            assert ws[:65536].max() == 0


def test_refusals(cuda_device):
    pool = Fp8Pool([20, 30], 2, 64, 16, seed=27, device=cuda_device)
    q = queries(2, 14, 64, 28, cuda_device)
    k, v, ks, vs, t, n = pool.args()
    for bad in ((q.float(), k, v, ks, vs, t, n), (q[:1], k, v, ks, vs, t, n),
                (q[:, :13], k, v, ks, vs, t, n), (q[..., :32], k, v, ks, vs, t, n),
                (q, k.view(torch.uint8), v, ks, vs, t, n), (q, k, v[:-1], ks, vs, t, n),
                (q, k, v, ks[:, :1], vs, t, n), (q, k, v, ks, vs.double(), t, n),
                (q, k, v, ks, vs, t.long(), n), (q, k, v, ks, vs, t, n.cpu())):
        with pytest.raises(AssertionError):
            paged_attention_decode_fp8(*bad, 0.125)
    with pytest.raises(_native.NativeLibraryError, match="group size 17"):
        paged_attention_decode_fp8(queries(2, 34, 64, 0, cuda_device), k, v, ks, vs, t, n, 0.125)
    odd = Fp8Pool([20], 2, 48, 16, seed=29, device=cuda_device)
    with pytest.raises(_native.NativeLibraryError, match="head_dim 48"):
        paged_attention_decode_fp8(queries(1, 2, 48, 0, cuda_device), *odd.args(), 0.125)
    wide = torch.zeros(pool.blocks, 16, 2, 72, dtype=torch.uint8, device=cuda_device).view(FP8)
    with pytest.raises(_native.NativeLibraryError, match="multiples of 16"):
        paged_attention_decode_fp8(q, wide[..., :64], v, ks, vs, t, n, 0.125)
    with pytest.raises(_native.NativeLibraryError, match="positive"):
        paged_attention_decode_fp8(q, k, v, ks, vs, t[:, :0], n, 0.125)
    assert paged_attention_decode_fp8(q[:0], k, v, ks, vs, t[:0], n[:0], 0.125).shape == (0, 14, 64)
