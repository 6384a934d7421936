"""A few tokens per sequence over the 8-bit pool: the calls of at most 64 (token, query head)
columns per kv head, 32 at head_dim 128, which have a kernel form of their own (needs an MI355X).

Values against the 64-bit oracle with its own bound per element; everything else bit by bit.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from _fp8_pool import FP8, Fp8Pool, int32, starts_of
from engine.kernels import _native
from engine.kernels.quantized_cache import paged_attention_prefill_fp8
from oracle import fp8_cache_oracle as oracle

pytestmark = pytest.mark.gpu

# Query heads, kv heads, head_dim, block size: block forms of 16 tokens and of any number, two
# and four blocks of columns, at head_dim 32 to 128.
SHAPES = [(14, 2, 64, 16), (14, 2, 64, 8), (8, 4, 64, 32), (4, 2, 32, 16), (26, 2, 32, 7), (8, 2, 128, 16),
          (12, 2, 128, 5)]


def queries(n, hq, d, seed, device):
    return torch.randn(n, hq, d, generator=torch.Generator().manual_seed(seed)).half().to(device)


def run(pool, q, new, scale, longest=None):
    longest = longest or max(new)
    assert longest * (q.shape[1] // pool.hkv) <= (64 if pool.d <= 64 else 32)
    return paged_attention_prefill_fp8(q, *pool.args(), int32(starts_of(new), pool.device), longest,
                                       scale)


def check(pool, q, new, scale):
    out = run(pool, q, new, scale)
    want, tol = oracle.attention(pool.state(), q.double().cpu().numpy(), pool.tables, pool.lens,
                                 starts_of(new), pool.bs, scale, bound=True)
    got = out.double().cpu().numpy()
    assert np.isfinite(got).all()
    off = np.abs(got - want)
    assert (off <= tol).all(), f"{(off / np.maximum(tol, 1e-30)).max():.3g} of the bound"
    return out


@pytest.mark.parametrize("lens", [[60, 130, 20], [60, 2600, 20]])
@pytest.mark.parametrize("hq,hkv,d,bs", SHAPES)
def test_nan_in_rows_that_are_not_seen(cuda_device, hq, hkv, d, bs, lens):
    """Behind the end, in unused blocks and their scales, and in later tokens of the same sequence:
    only the rows that see a NaN become NaN."""
    new = [4, 3, 2]
    pool = Fp8Pool(lens, hkv, d, bs, seed=9, device=cuda_device)
    q, g = queries(9, hq, d, 10, cuda_device), hq // hkv
    used = np.zeros((pool.blocks, bs), dtype=bool)
    for b, n in enumerate(lens):
        for p in range(n):
            used[pool.tables[b, p // bs], p % bs] = True
    base = check(pool, q, new, 0.125)
    hole = torch.from_numpy(~used).to(cuda_device)
    for cache in (pool.dk, pool.dv):
        cache.view(torch.uint8)[hole] = 0xff
    unused = torch.from_numpy(~used.any(axis=1)).to(cuda_device)
    pool.dks[unused] = float("nan")
    pool.dvs[unused] = float("inf")
    assert torch.equal(run(pool, q, new, 0.125), base)
    last = slice((hkv - 1) * g, hq)
    # The sequences' tokens at a position, kv head hkv - 1: which rows see it.
    for b, pos, first in ((0, 58, 2), (0, 59, 3), (0, 56, 0), (0, 3, 0), (1, lens[1] - 2, 5), (1, 64, 4),
                          (2, 19, 8)):
        end = starts_of(new)[b + 1]
        for cache, at, code in ((pool.dv, 5, 0x7f), (pool.dk, d - 1, 0xff), (pool.dv, d - 1, 0xff)):
            place = (pool.tables[b, pos // bs], pos % bs, hkv - 1, at)
            was = cache.view(torch.uint8)[place].clone()
            cache.view(torch.uint8)[place] = code
            out = run(pool, q, new, 0.125)
            assert out[first:end, last].isnan().any(dim=2).all(), (b, pos, at)
            out[first:end, last] = base[first:end, last]
            assert torch.equal(out, base), (b, pos, at)
            cache.view(torch.uint8)[place] = was


@pytest.mark.parametrize("hq,hkv,d,bs", SHAPES)
def test_tables_and_lengths_out_of_range(cuda_device, hq, hkv, d, bs):
    """Contexts shorter than their new rows (zeros), longer than the table (cut), bad block ids
    (clamped)."""
    pool = Fp8Pool([64, 64, 30, 12], hkv, d, bs, seed=11, device=cuda_device)
    pool.tables[0, 1] = -7
    pool.tables[1, 0] = pool.blocks + 5
    pool.dt = torch.from_numpy(pool.tables).to(cuda_device)
    pool.lens = [64, 5000, 3, -2]
    pool.dl = int32(pool.lens, cuda_device)
    new = [4, 3, 4, 2]
    out = check(pool, queries(13, hq, d, 12, cuda_device), new, 0.125)
    assert not out[7].any() and out[8:11].any() and not out[11:].any()


@pytest.mark.parametrize("longest", [40, 3000])
@pytest.mark.parametrize("hq,hkv,d,bs", SHAPES)
def test_cache_scales_of_the_whole_range(cuda_device, hq, hkv, d, bs, longest):
    pool = Fp8Pool([longest, 33], hkv, d, bs, seed=7, device=cuda_device)
    g = torch.Generator().manual_seed(1)
    pool.dvs.copy_(torch.exp2(torch.randint(-15, 8, pool.v_scale.shape, generator=g).float()))
    pool.dks.copy_(torch.exp2(torch.randint(-15, -6, pool.k_scale.shape, generator=g).float()))
    check(pool, queries(7, hq, d, 8, cuda_device), [3, 4], 0.125)


@pytest.mark.parametrize("scale", [4.0, 1e-3])
@pytest.mark.parametrize("hq,hkv,d,bs", SHAPES)
def test_peaked_and_flat(cuda_device, hq, hkv, d, bs, scale):
    pool = Fp8Pool([2500, 40, 3], hkv, d, bs, seed=5, device=cuda_device)
    check(pool, queries(9, hq, d, 6, cuda_device), [4, 2, 3], scale)


@pytest.mark.parametrize("hq,hkv,d,bs", SHAPES)
def test_rows_of_no_sequence_and_past_the_longest_are_left(cuda_device, hq, hkv, d, bs):
    """Through the C ABI, whose output is the caller's: rows before the first sequence, behind the
    last, and past max_query_len of a sequence."""
    pool = Fp8Pool([70, 2100, 5], hkv, d, bs, seed=13, device=cuda_device)
    q = queries(12, hq, d, 14, cuda_device)
    starts = [2, 4, 9, 10]
    out = torch.full_like(q, 7.0)
    lib, st = _native.load(), _native.strides_of
    dev_starts = int32(starts, cuda_device)
    sizes = (3, hq, hkv, d, bs, pool.dt.shape[1], 3)
    nbytes = lib.pa_prefill_attention_fp8_workspace_bytes(*sizes)
    ws = torch.zeros(max(nbytes, 1), dtype=torch.uint8, device=cuda_device)
    status = lib.pa_prefill_attention_fp8(
        q.data_ptr(), st(q), pool.dk.data_ptr(), st(pool.dk), pool.dv.data_ptr(), st(pool.dv),
        pool.dks.data_ptr(), st(pool.dks), pool.dvs.data_ptr(), st(pool.dvs), pool.dt.data_ptr(),
        st(pool.dt), pool.dl.data_ptr(), dev_starts.data_ptr(), 3, out.data_ptr(), st(out), 3, 12, hq,
        hkv, d, bs, pool.blocks, pool.dt.shape[1], 0.125, ws.data_ptr(), nbytes,
        _native.stream_handle(cuda_device))
    assert status == _native.PA_OK
    kept = [0, 1, 7, 8, 10, 11]
    assert (out[kept] == 7).all()
    want, tol = oracle.attention(pool.state(), q[2:10].double().cpu().numpy(), pool.tables, pool.lens,
                                 [0, 2, 7, 8], bs, 0.125, bound=True)
    off = np.abs(out[2:10].double().cpu().numpy() - want)
    written = [0, 1, 2, 3, 4, 7]
    assert (off[written] <= tol[written]).all()
    assert not ws[:65536].any()


def test_offsets_past_32_bits(cuda_device):
    blocks, bs, hkv, d = 2 ** 16 + 9, 16, 32, 128  # 65,536 codes a block
    small = Fp8Pool([45], hkv, d, bs, seed=21, device=cuda_device)
    q = queries(4, 64, d, 22, cuda_device)
    base = check(small, q, [4], d ** -0.5)
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
    starts = int32([0, 4], cuda_device)
    for most in (4, 40):  # this form, and the one for prompts
        out = paged_attention_prefill_fp8(q, *big, int32([ids], cuda_device), small.dl, starts, most,
                                          d ** -0.5)
        want = paged_attention_prefill_fp8(q, *small.args(), starts, most, d ** -0.5)
        assert torch.equal(out, want)
    assert torch.equal(run(small, q, [4], d ** -0.5), base)


@torch.inference_mode()  # as every capture among these tests: torch's generator state may be one of it
@pytest.mark.parametrize("hq,hkv,d,bs", SHAPES)
def test_strides_and_graphs(cuda_device, hq, hkv, d, bs):
    """Query slices, heads-first values, transposed scales; two captured calls replayed at once on
    two streams, eager calls beside them."""
    lens, new = [90, 5000, 16], [4, 3, 1]
    pool = Fp8Pool(lens, hkv, d, bs, seed=15, device=cuda_device)
    q = queries(8, hq, d, 16, cuda_device)
    base = check(pool, q, new, 0.125)
    wide = torch.zeros(8, hq, 3, d, dtype=torch.float16, device=cuda_device)
    wide[:, :, 1] = q
    pool.dv = pool.dv.view(torch.uint8).transpose(1, 2).contiguous().view(FP8).transpose(1, 2)
    pool.dks = pool.dks.t().contiguous().t()
    assert torch.equal(run(pool, wide[:, :, 1], new, 0.125), base)
    starts = int32(starts_of(new), cuda_device)
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for part in (q, wide[:, :, 1]):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(paged_attention_prefill_fp8(part, *pool.args(), starts, 4, 0.125))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for seed in range(4):
        x = queries(8, hq, d, 40 + seed, cuda_device)
        q.copy_(x)
        wide[:, :, 1] = x
        want = run(pool, q, new, 0.125)
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = run(pool, q, new, 0.125)
        torch.cuda.synchronize()
        for out in (*outs, eager):
            assert torch.equal(out, want)
    for key, ws in _native._workspaces.items():
        if key[2] == _native.WS_PREFILL:
            assert ws[:65536].max() == 0
