"""Attention over the 8-bit pool and its read where values, scales or counts are unusual (needs an
MI355X). Outputs are compared bit by bit, or for being NaN: no tolerance is used.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from _fp8_pool import Fp8Pool, int32, starts_of
from engine.kernels import _native
from engine.kernels.quantized_cache import (
    paged_attention_decode_fp8,
    paged_attention_prefill_fp8,
    paged_kv_read_fp8,
)

pytestmark = pytest.mark.gpu


def queries(n, hq, d, seed, device, std=1.0):
    x = torch.randn(n, hq, d, generator=torch.Generator().manual_seed(seed)) * std
    return x.half().to(device)


def attend(pool, q, new, scale, longest=None):
    """`new` tokens per sequence through the several-token call (of up to `longest`), or None: the
    decode call."""
    if new is None:
        return paged_attention_decode_fp8(q, *pool.args(), scale)
    return paged_attention_prefill_fp8(q, *pool.args(), int32(starts_of(new), pool.device),
                                       longest or max(new), scale)


@pytest.mark.parametrize("new", [None, [4], [40], [300]])
@pytest.mark.parametrize("spoiled", [31, 1000, 1024, 1536, 6144, 8600])
def test_nan_in_the_first_keys_only(cuda_device, new, spoiled):
    """Enough of them that whole splits of the keys see nothing else: every row sees them and is
    NaN, and no row of the other kv head."""
    pool = Fp8Pool([9000], 2, 64, 16, seed=1, device=cuda_device)
    q = queries(sum(new or [1]), 14, 64, 2, cuda_device)
    base = attend(pool, q, new, 0.125)
    pos = np.arange(spoiled)
    pool.dk.view(torch.uint8)[pool.tables[0, pos // 16], pos % 16, 1] = 0x7f
    out = attend(pool, q, new, 0.125)
    assert torch.equal(out[:, :7], base[:, :7]) and base.isfinite().all()
    assert out[:, 7:].isnan().all()


def sharp(pool, q, scale):
    """Where one score lies so far above a row's others that fp32 sums of the products cannot
    mistake it and the others' weights are 0 -- [sequences, heads], nearly everywhere -- and that
    key's V row, which is then the output, exactly."""
    rows, where = [], []
    k, v = ((getattr(pool, c).double() * getattr(pool, c + "_scale").double()[:, None, :, None])
            for c in ("k", "v"))
    group = q.shape[1] // pool.hkv
    for b, n in enumerate(pool.lens):
        ids = torch.from_numpy(pool.tables[b].astype(np.int64))
        keys, values = (x[ids].reshape(-1, pool.hkv, pool.d)[:n].repeat_interleave(group, 1).transpose(0, 1)
                        for x in (k, v))
        x = q[b].double().cpu()[:, :, None]
        top = (keys @ x)[..., 0].mul(scale).topk(min(2, n), dim=1)
        size = (keys.abs() @ x.abs()).amax() * abs(scale)
        far = 100 + 2 * (pool.d + 8) * size * 2.0 ** -24
        where.append(top.values[:, 0] - top.values[:, -1] > (far if n > 1 else -1))
        rows.append(values[torch.arange(len(values)), top.indices[:, 0]])
    where = torch.stack(where)
    assert where.double().mean() > 0.98
    return where, torch.stack(rows).half()


@pytest.mark.parametrize("seqs", [2, 300])
@pytest.mark.parametrize("several,scale,hq,hkv,d,bs", [
    (several, scale, *shape) for several, scale in [(False, 0.125), (False, -0.125), (False, 16.0), (True, 16.0)]
    for shape in [(14, 2, 64, 16), (4, 2, 64, 8), (8, 2, 128, 16), (3, 1, 256, 16)][:3 if several else 4]])
def test_scores_of_many_millions(cuda_device, several, scale, hq, hkv, d, bs, seqs):
    """Scores beyond what fp32 holds to one unit: the largest one's weight is still 1."""
    lens = [1 + (97 * i) % 290 for i in range(seqs)]
    lens[1] = 2500
    pool = Fp8Pool(lens, hkv, d, bs, seed=hq + d, device=cuda_device)
    pool.k_scale = pool.k_scale * 2.0 ** 12
    pool.dks = pool.k_scale.to(cuda_device)
    q = queries(seqs, hq, d, 4, cuda_device, std=2000.0)
    where, rows = sharp(pool, q, scale)
    out = attend(pool, q, [1] * seqs if several else None, scale).cpu()
    assert out.isfinite().all() and torch.equal(out[where], rows[where])


@pytest.mark.parametrize("seqs", [2, 300])
@pytest.mark.parametrize("hq,hkv,d,bs", [(14, 2, 64, 16), (4, 2, 32, 8), (8, 2, 128, 16), (3, 1, 256, 16)])
def test_scores_of_many_millions_in_a_call_for_prompts(cuda_device, hq, hkv, d, bs, seqs):
    """The same in the kernel that takes calls of up to 100 tokens per sequence."""
    lens = [1 + (97 * i) % 290 for i in range(seqs)]
    lens[1] = 2500
    pool = Fp8Pool(lens, hkv, d, bs, seed=hq + d, device=cuda_device)
    pool.k_scale = pool.k_scale * 2.0 ** 12
    pool.dks = pool.k_scale.to(cuda_device)
    q = queries(seqs, hq, d, 4, cuda_device, std=2000.0)
    where, rows = sharp(pool, q, 64.0)
    out = attend(pool, q, [1] * seqs, 64.0, longest=100).cpu()
    assert out.isfinite().all() and torch.equal(out[where], rows[where])


@pytest.mark.parametrize("d", [64, 5])
def test_read_of_no_sequence_through_the_c_abi(cuda_device, d):
    """All rows are rows of no sequence: zeros, whatever the other arguments are."""
    lib, st = _native.load(), _native.strides_of
    pool = Fp8Pool([20], 2, d, 16, seed=3, device=cuda_device)
    starts = int32([0], cuda_device)
    real = (pool.dk.data_ptr(), st(pool.dk), pool.dv.data_ptr(), st(pool.dv), pool.dks.data_ptr(),
            st(pool.dks), pool.dvs.data_ptr(), st(pool.dvs), pool.dt.data_ptr(), st(pool.dt),
            pool.dl.data_ptr(), starts.data_ptr())
    for args, bs, blocks, width in ((real, 16, pool.blocks, pool.dt.shape[1]), ((None,) * 12, 0, 0, 0)):
        wide = [torch.full((40, 2, d), 7.0, dtype=torch.float16, device=cuda_device) for _ in range(2)]
        rows = [x[1:38] for x in wide]
        status = lib.pa_kv_read_fp8(
            *args, rows[0].data_ptr(), st(rows[0]), rows[1].data_ptr(), st(rows[1]), 0, 37, 2, d, bs,
            blocks, width, _native.stream_handle(cuda_device))
        assert status == _native.PA_OK
        for x in wide:
            assert not x[1:38].any() and (x[:1] == 7).all() and (x[38:] == 7).all()


@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (4, 2, 32), (8, 2, 128), (3, 1, 256)])
@pytest.mark.parametrize("bs", [5, 8, 16, 32, 48])
def test_scales_count_by_their_exponent(cuda_device, hq, hkv, d, bs):
    """A pool whose scales are no powers of two gives what the next lower powers give, whatever the
    block size and the call."""
    lens = [300, 2, 2500]
    pool = Fp8Pool(lens, hkv, d, bs, seed=5, device=cuda_device)
    calls = [(None, None), ([2, 1, 3], 4), ([2, 1, 3], 100)]
    qs = [queries(sum(new or [1] * 3), hq, d, 6, cuda_device) for new, _ in calls]
    base = [attend(pool, q, new, 0.125, most) for q, (new, most) in zip(qs, calls)]
    starts = int32(starts_of(lens), cuda_device)
    rows = paged_kv_read_fp8(*pool.args(), starts, sum(lens))
    pool.dks, pool.dvs = pool.dks * 1.5, pool.dvs * 1.9375
    for q, (new, most), want in zip(qs, calls, base):
        assert torch.equal(attend(pool, q, new, 0.125, most), want)
    for got, want in zip(paged_kv_read_fp8(*pool.args(), starts, sum(lens)), rows):
        assert torch.equal(got, want)
