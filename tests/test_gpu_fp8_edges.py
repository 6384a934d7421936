"""Attention over the 8-bit pool and its read where values, scales or counts are unusual (needs an
MI355X). Outputs are compared bit by bit, or for being NaN: no tolerance is used.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from _fp8_pool import Fp8Pool, int32, starts_of
from engine.kernels.quantized_cache import paged_attention_decode_fp8, paged_attention_prefill_fp8

pytestmark = pytest.mark.gpu


def queries(n, hq, d, seed, device, std=1.0):
    x = torch.randn(n, hq, d, generator=torch.Generator().manual_seed(seed)) * std
    return x.half().to(device)


def attend(pool, q, new, scale):
    """`new` tokens per sequence through the several-token call, or None: the decode call."""
    if new is None:
        return paged_attention_decode_fp8(q, *pool.args(), scale)
    return paged_attention_prefill_fp8(q, *pool.args(), int32(starts_of(new), pool.device), max(new),
                                       scale)


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
