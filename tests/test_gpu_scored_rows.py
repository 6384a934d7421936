"""Rows of the scored prefill past max_query_len (needs an MI355X)."""
from __future__ import annotations

import pytest
import torch

from _scored import Pool, slopes_of
from engine.kernels import _native
from engine.kernels.scored_attention import paged_attention_prefill_scored

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,hkv,d", [(14, 2, 64), (8, 2, 128), (3, 3, 32), (4, 1, 256)])
@pytest.mark.parametrize("most", [1, 5, 31, 60, 2000])
def test_rows_past_the_longest_are_left_alone(cuda_device, heads, hkv, d, most):
    lens, new = [1500, 90, 40], [70, 61, 3]
    pool = Pool(lens, hkv, d, 16, cuda_device)
    q = pool.queries(sum(new), heads)
    loc, slopes = pool.ints([0, 70, 131, 134]), slopes_of(heads, cuda_device)
    args = (pool.k, pool.v, pool.tables, pool.seq_lens, loc)
    want = paged_attention_prefill_scored(q, *args, 70, 0.125, 9.0, slopes, 50)
    lib, st = _native.load(), _native.strides_of
    out = torch.full_like(q, 7.0)
    width = pool.tables.shape[1]
    nbytes = lib.pa_prefill_attention_scored_workspace_bytes(3, heads, hkv, d, 16, width, most, 50, 0)
    ws = torch.zeros(max(nbytes, 16), dtype=torch.uint8, device=cuda_device)
    status = lib.pa_prefill_attention_scored_f16(
        q.data_ptr(), st(q), pool.k.data_ptr(), st(pool.k), pool.v.data_ptr(), st(pool.v),
        pool.tables.data_ptr(), st(pool.tables), pool.seq_lens.data_ptr(), loc.data_ptr(), most,
        out.data_ptr(), st(out), 3, sum(new), heads, hkv, d, 16, pool.blocks, width, 0.125, 9.0,
        slopes.data_ptr(), 1, 50, None, None, ws.data_ptr(), nbytes, _native.stream_handle(q.device))
    _native.check(status, "pa_prefill_attention_scored_f16")
    at = 0
    for n in new:
        # (Splits of the keys depend on max_query_len: to two roundings of values up to 4.)
        assert (out[at:at + min(n, most)].float() - want[at:at + min(n, most)].float()).abs().max() < 8e-3
        assert (out[at + min(n, most):at + n] == 7).all()
        at += n
