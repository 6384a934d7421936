"""Writing the 8-bit pool and reading it back, against the 64-bit oracle (needs an MI355X).

Codes, scales and values are compared exactly: with power-of-two scales a value is rounded
once, to nearest even, on both sides. The whole pool is compared, so a write outside the
slots shows.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from engine.kernels import _native
from engine.kernels.quantized_cache import paged_kv_read_fp8, paged_kv_write_fp8
from oracle import fp8_cache_oracle as oracle
from _fp8_pool import Fp8Pool, int32, starts_of

pytestmark = pytest.mark.gpu


def rows(tokens, hkv, d, seed, device, wide=True):
    """fp16 rows whose channels differ in width by orders of magnitude."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, hkv, d, generator=g)
    if wide:
        x = x * torch.exp(1.5 * torch.randn(tokens, hkv, d, generator=g))
    return x.half().to(device)


def same_state(pool, want):
    got = pool.state()
    for name in want:
        assert np.array_equal(got[name], want[name], equal_nan=True), name


def check_write(pool, key, value, new, one=False):
    want = pool.oracle()
    starts = starts_of(new)
    oracle.write(want, key.double().cpu().numpy(), value.double().cpu().numpy(), pool.tables,
                 pool.lens, starts, pool.bs)
    call = (key, value, *pool.args())
    if not one:
        call += (int32(starts, pool.device),)
    for _ in range(2):  # repeated, nothing changes
        paged_kv_write_fp8(*call)
        same_state(pool, want)


@pytest.mark.parametrize("hkv,d,bs", [(2, 64, 16), (8, 128, 16), (4, 128, 32), (7, 128, 8), (2, 32, 16),
                                      (2, 256, 16), (3, 40, 5), (1, 24, 1), (2, 20, 16), (1, 1, 7)])
def test_one_row_per_sequence(cuda_device, hkv, d, bs):
    lens = [1, 2, bs, bs + 1, 3 * bs, 77, 500, 0] + list(range(30, 50))
    pool = Fp8Pool(lens, hkv, d, bs, seed=hkv * 1000 + d + bs, device=cuda_device)
    n = len(lens)
    check_write(pool, rows(n, hkv, d, 1, cuda_device), rows(n, hkv, d, 2, cuda_device), [1] * n,
                one=True)


@pytest.mark.parametrize("hkv,d,bs", [(2, 64, 16), (8, 128, 16), (4, 128, 32), (7, 128, 8), (2, 256, 64),
                                      (3, 40, 5), (1, 24, 1), (2, 20, 16), (1, 8, 300)])
def test_several_rows_per_sequence(cuda_device, hkv, d, bs):
    """Whole prompts, chunks that begin and end inside blocks, drafts, nothing; more sequences
    than one step of the search takes."""
    lens = [100, 1, 333, 64, 5 * bs, 40] + [20 + i for i in range(90)]
    new = [100, 1, 130, 0, 2 * bs, 7] + [i % 6 for i in range(90)]
    pool = Fp8Pool(lens, hkv, d, bs, seed=hkv + d + bs, device=cuda_device)
    n = sum(new)
    check_write(pool, rows(n, hkv, d, 3, cuda_device), rows(n, hkv, d, 4, cuda_device), new)


def test_special_values(cuda_device):
    """NaN stays NaN and does not set the scale, infinities are the largest value, all-zero and
    all-NaN rows take the smallest scale."""
    lens, new = [40, 16, 16, 33], [40, 16, 16, 1]
    pool = Fp8Pool(lens, 2, 64, 16, seed=5, device=cuda_device)
    key = rows(sum(new), 2, 64, 6, cuda_device)
    key[3, 0, 5] = float("nan")
    key[20, 1, 9] = float("inf")
    key[21, 0, 0] = -65504.0
    key[35, 0, 3] = 61440.0
    key[36, 1, 3] = 57376.0
    key[40:56] = 0.0
    key[56:72] = float("nan")
    key[72] = 2.0 ** -24
    value = -key
    value[72] = -float("inf")
    check_write(pool, key, value, new)
    got = pool.state()
    assert np.isnan(got["k"]).sum() == 1 + 16 * 2 * 64
    assert np.abs(got["v"][np.isfinite(got["v"])]).max() <= 448


@pytest.mark.parametrize("vec", [True, False])
def test_growing_scales_recode_the_rows_before(cuda_device, vec):
    """One row at a time, each larger than all before, over block boundaries."""
    d = 64 if vec else 36
    n = 40
    pool = Fp8Pool([n], 2, d, 16, seed=8, device=cuda_device)
    want = pool.oracle()
    x = rows(n, 2, d, 9, cuda_device, wide=False)
    x = (x.float() * torch.exp2(torch.arange(n, device=cuda_device).float() / 2 - 12)[:, None, None]).half()
    for i in range(n):
        lens = int32([i + 1], cuda_device)
        paged_kv_write_fp8(x[i:i + 1], -x[i:i + 1], *pool.args()[:5], lens)
        oracle.write(want, x[i:i + 1].double().cpu().numpy(), -x[i:i + 1].double().cpu().numpy(),
                     pool.tables, [i + 1], [0, 1], 16)
        same_state(pool, want)


def test_tokens_taken_back(cuda_device):
    """Drafts written, some rejected, other rows written over them."""
    pool = Fp8Pool([20, 35], 2, 64, 16, seed=10, device=cuda_device)
    want = pool.oracle()
    for lens, new, seed in (([20, 35], [5, 5], 1), ([17, 33], [1, 2], 2), ([21, 38], [4, 5], 3)):
        x, y = rows(sum(new), 2, 64, seed, cuda_device), rows(sum(new), 2, 64, seed + 9, cuda_device)
        paged_kv_write_fp8(x, y, *pool.args()[:5], int32(lens, cuda_device),
                           int32(starts_of(new), cuda_device))
        oracle.write(want, x.double().cpu().numpy(), y.double().cpu().numpy(), pool.tables, lens,
                     starts_of(new), 16)
        same_state(pool, want)


def test_rows_without_a_slot(cuda_device):
    """Lengths below the row count, past the table, and block ids outside the pool."""
    pool = Fp8Pool([40, 64, 50, 30], 2, 64, 16, seed=11, device=cuda_device)
    pool.tables[1, 1] = -3
    pool.tables[2, 3] = pool.blocks
    pool.dt = torch.from_numpy(pool.tables).to(cuda_device)
    pool.lens = [3, 70, 50, -4]
    pool.dl = int32(pool.lens, cuda_device)
    new = [8, 70, 50, 2]
    check_write(pool, rows(130, 2, 64, 12, cuda_device), rows(130, 2, 64, 13, cuda_device), new)
    key, value = paged_kv_read_fp8(*pool.args(), int32(starts_of(new), cuda_device), 130)
    want = oracle.read(pool.state(), pool.tables, pool.lens, starts_of(new), 16, 130)
    assert np.array_equal(key.cpu().double().numpy(), want[0])
    assert np.array_equal(value.cpu().double().numpy(), want[1])


@pytest.mark.parametrize("starts", [[4, 2, 9, 9], [-5, 3, 3, 99], [7, 7, 7, 7], [9, 0, 0, 0]])
def test_starts_out_of_order_or_range_stay_in_bounds(cuda_device, starts):
    """Such a call's rows are undefined, but nothing outside the pool's blocks is touched."""
    pool = Fp8Pool([20, 20, 20], 2, 64, 16, seed=14, device=cuda_device)
    guard = torch.full((3 * pool.dk.numel(),), 0x55, dtype=torch.uint8, device=cuda_device)
    inner = guard[pool.dk.numel():2 * pool.dk.numel()].view(torch.float8_e4m3fn)
    pool.dk = inner.view(pool.dk.shape)
    x = rows(9, 2, 64, 15, cuda_device)
    paged_kv_write_fp8(x, x, *pool.args(), int32(starts, cuda_device))
    paged_kv_read_fp8(*pool.args(), int32(starts, cuda_device), 9)
    torch.cuda.synchronize()
    n = pool.dk.numel()
    assert (guard[:n] == 0x55).all() and (guard[2 * n:] == 0x55).all()


def test_strided_sources_pools_and_scales(cuda_device):
    """Slices of a merged projection, an inner stride, a pool inside a larger one, odd bases."""
    lens, new = [30, 50], [11, 50]
    n = sum(new)
    big = rows(n, 6, 128, 16, cuda_device)
    for key, value in ((big[:, :2, :64], big[:, 2:4, 64:]), (big[:, ::3, ::2], big[:, 1::3, 1::2]),
                       (big[:, :2, 3:67], big[:, 4:, :64])):
        pool = Fp8Pool(lens, 2, 64, 16, seed=17, device=cuda_device)
        wide = torch.zeros(pool.blocks, 16, 2, 200, dtype=torch.uint8, device=cuda_device)
        for lo in (64, 7):
            pool.dk = wide.view(torch.float8_e4m3fn)[..., lo:lo + 64]
            pool.dk.view(torch.uint8).copy_(pool.k.view(torch.uint8).to(cuda_device))
            pool.dv = pool.v.to(cuda_device)
            pool.dks = pool.k_scale.t().contiguous().to(cuda_device).t()
            pool.dvs = pool.v_scale.to(cuda_device)
            check_write(pool, key, value, new)
            got = paged_kv_read_fp8(*pool.args(), int32(starts_of(new), cuda_device), n)
            want = oracle.read(pool.state(), pool.tables, lens, starts_of(new), 16, n)
            for a, b in zip(got, want):
                assert np.array_equal(a.cpu().double().numpy(), b)


@pytest.mark.parametrize("hkv,d,bs", [(2, 64, 16), (8, 128, 16), (4, 128, 32), (7, 128, 8), (2, 256, 64),
                                      (3, 40, 5), (1, 24, 1), (2, 20, 16), (1, 16, 300)])
def test_read(cuda_device, hkv, d, bs):
    """Whole contexts, tails, nothing; rows before the first and behind the last sequence are zeros."""
    lens = [100, 1, 333, 64, 0, 5 * bs, 40] + [20 + i for i in range(90)]
    new = [100, 1, 130, 0, 0, 2 * bs, 7] + [i % 6 for i in range(90)]
    pool = Fp8Pool(lens, hkv, d, bs, seed=hkv + d, device=cuda_device, spread=1.6)
    starts = [s + 5 for s in starts_of(new)]
    total = starts[-1] + 9
    key, value = paged_kv_read_fp8(*pool.args(), int32(starts, cuda_device), total)
    want = oracle.read(pool.oracle(), pool.tables, lens, starts, bs, total)
    assert np.array_equal(key.cpu().double().numpy(), want[0])
    assert np.array_equal(value.cpu().double().numpy(), want[1])
    assert key[:5].abs().max() == 0 and value[-9:].abs().max() == 0


def test_read_of_every_code_and_scale(cuda_device):
    """All 256 codes at every scale: an fp16 number each (240 * 2^8 is the largest written)."""
    pool = Fp8Pool([24 * 16], 1, 256, 16, seed=1, device=cuda_device)
    codes = torch.arange(256, dtype=torch.uint8).expand(pool.blocks, 16, 1, 256).contiguous()
    pool.k = codes.view(torch.float8_e4m3fn)
    pool.dk = pool.k.to(cuda_device)
    for j, block in enumerate(pool.tables[0]):
        pool.k_scale[block] = 2.0 ** (j - 15)
    pool.dks = pool.k_scale.to(cuda_device)
    key, _ = paged_kv_read_fp8(*pool.args(), int32([0, 384], cuda_device), 384)
    want = (pool.k.float() * pool.k_scale[:, None, :, None])[torch.from_numpy(pool.tables[0]).long()]
    want = want.reshape(384, 1, 256)
    got = key.cpu().float()
    exact = want.isnan() | (want.abs() <= 61440)
    assert exact.float().mean() > 0.99
    assert torch.equal(got[exact].nan_to_num(7e6), want[exact].nan_to_num(7e6))


def test_offsets_past_32_bits(cuda_device):
    """A pool of more than 2^32 codes: the last block's rows."""
    blocks, bs, hkv, d = 2 ** 16 + 9, 16, 32, 128  # 65,536 codes a block
    pool = Fp8Pool([35], hkv, d, bs, seed=2, device=cuda_device)
    k = torch.zeros(blocks, bs, hkv, d, dtype=torch.uint8, device=cuda_device)
    scale = torch.ones(blocks, hkv, device=cuda_device)
    v, vscale = k.clone(), scale.clone()
    ids = torch.tensor([[blocks - 1, 3, blocks - 2]], dtype=torch.int32, device=cuda_device)
    x = rows(35, hkv, d, 3, cuda_device)
    args = (k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), scale, vscale, ids, pool.dl)
    starts = int32([0, 35], cuda_device)
    paged_kv_write_fp8(x, -x, *args, starts)
    key, value = paged_kv_read_fp8(*args, starts, 35)
    assert torch.equal(key, -value)
    small = Fp8Pool([35], hkv, d, bs, seed=2, device=cuda_device)
    paged_kv_write_fp8(x, -x, *small.args(), starts)
    want, _ = paged_kv_read_fp8(*small.args(), starts, 35)
    assert torch.equal(key, want)


@torch.inference_mode()  # as every capture among these tests: torch's generator state may be one of it
def test_on_another_stream_and_in_a_graph(cuda_device):
    """A captured write and read, replayed on changing rows with eager work between."""
    lens, new = [50, 20, 128], [3, 20, 1]
    pool = Fp8Pool(lens, 2, 64, 16, seed=20, device=cuda_device)
    starts = int32(starts_of(new), cuda_device)
    x, y = rows(24, 2, 64, 0, cuda_device), rows(24, 2, 64, 1, cuda_device)
    paged_kv_write_fp8(x, y, *pool.args(), starts)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            paged_kv_write_fp8(x, y, *pool.args(), starts)
            key, value = paged_kv_read_fp8(*pool.args(), starts, 24)
    for seed in range(3):
        x.copy_(rows(24, 2, 64, 30 + seed, cuda_device))
        y.copy_(rows(24, 2, 64, 40 + seed, cuda_device))
        torch.cuda.synchronize()
        want = pool.state()
        graph.replay()
        torch.cuda.synchronize()
        oracle.write(want, x.double().cpu().numpy(), y.double().cpu().numpy(), pool.tables, lens,
                     starts_of(new), 16)
        same_state(pool, want)
        rk, rv = oracle.read(want, pool.tables, lens, starts_of(new), 16, 24)
        assert np.array_equal(key.cpu().double().numpy(), rk)
        assert np.array_equal(value.cpu().double().numpy(), rv)


def test_refusals(cuda_device):
    pool = Fp8Pool([20, 30], 2, 64, 16, seed=21, device=cuda_device)
    x = rows(2, 2, 64, 0, cuda_device)
    k, v, ks, vs, t, n = pool.args()
    starts = int32([0, 1, 2], cuda_device)
    good = dict(key=x, value=x, k_cache=k, v_cache=v, k_scale=ks, v_scale=vs, block_tables=t,
                seq_lens=n)
    for bad in (dict(key=x.float()), dict(value=x[:1]), dict(key=x[..., :32], value=x[..., :32]),
                dict(k_cache=k.view(torch.uint8)), dict(k_cache=k[:, :8]), dict(k_scale=ks[:-1]),
                dict(v_scale=vs.half()), dict(block_tables=t.long()), dict(seq_lens=n.cpu()),
                dict(seq_lens=n[:1]), dict(block_tables=t[:1]), dict(key=x[:1], value=x[:1]),
                dict(query_start_loc=starts[:2]), dict(query_start_loc=starts.long())):
        with pytest.raises(AssertionError):
            paged_kv_write_fp8(**{**good, **bad})
    with pytest.raises(_native.NativeLibraryError, match="stride"):
        paged_kv_write_fp8(**{**good, "k_cache": k.transpose(1, 3).contiguous().transpose(1, 3)})
    with pytest.raises(_native.NativeLibraryError, match="positive"):
        paged_kv_write_fp8(**{**good, "block_tables": t[:, :0]})
    with pytest.raises(AssertionError):
        paged_kv_read_fp8(*pool.args(), starts, -1)
    with pytest.raises(AssertionError):
        paged_kv_read_fp8(*pool.args(), starts.cpu(), 2)
    # Nothing to do.
    paged_kv_write_fp8(x[:0], x[:0], k, v, ks, vs, t[:0], n[:0])
    paged_kv_write_fp8(x[:0], x[:0], k, v, ks, vs, t, n, int32([0, 0, 0], cuda_device))
    assert paged_kv_read_fp8(k, v, ks, vs, t[:0], n[:0], starts[:1], 3)[0].abs().max() == 0
    assert paged_kv_read_fp8(*pool.args(), starts, 0)[0].shape == (0, 2, 64)
    same_state(pool, pool.oracle())
