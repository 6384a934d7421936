"""Prefill attention with capped, biased and masked scores against the 64-bit oracle (needs an MI355X)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from _scored import Pool, check_prefill, slopes_of
from engine.kernels import _native
from engine.kernels.paged_attention import paged_attention_prefill
from engine.kernels.scored_attention import paged_attention_prefill_scored

pytestmark = pytest.mark.gpu

FORMS = [dict(softcap=20.0), dict(bias=True), dict(window=100), dict(softcap=5.0, bias=True, window=33)]


def documents(lens, new, size, seed=0):
    """First key of each row's document."""
    rng = np.random.default_rng(seed)
    out = []
    for n, k in zip(lens, new):
        cuts = np.unique(np.concatenate([[0], rng.integers(0, n, max(1, n // size))]))
        pos = np.arange(n - k, n)
        out.append(cuts[np.searchsorted(cuts, pos, side="right") - 1])
    return np.concatenate(out)


def prefixes(lens, new, sizes):
    """End of each row's keys where the first sizes[b] tokens are seen as a whole."""
    return np.concatenate([np.maximum(np.arange(n - k + 1, n + 1), s) for n, k, s in zip(lens, new, sizes)])


@pytest.mark.parametrize("heads,hkv,d", [(14, 2, 64), (32, 8, 128), (4, 4, 64), (4, 2, 32), (16, 2, 256),
                                         (16, 1, 64), (12, 1, 32)])
@pytest.mark.parametrize("bs", [16, 32, 5])
def test_shapes(cuda_device, heads, hkv, d, bs):
    lens, new = [1, 40, 150, 129, 64], [1, 7, 150, 64, 2]
    pool = Pool(lens, hkv, d, bs, cuda_device, seed=d + bs)
    q = pool.queries(sum(new), heads)
    slopes = slopes_of(heads, cuda_device)
    for f in FORMS:
        f = dict(f)
        check_prefill(pool, q, new, d ** -0.5, slopes=slopes if f.pop("bias", False) else None, **f)
    check_prefill(pool, q, new, d ** -0.5, starts=documents(lens, new, 20))
    check_prefill(pool, q, new, d ** -0.5, ends=prefixes(lens, new, [1, 39, 100, 129, 5]), slopes=slopes)


@pytest.mark.parametrize("heads,hkv,d", [(14, 2, 64), (8, 2, 128)])
def test_long_prompts(cuda_device, heads, hkv, d):
    """Column blocks of every form, key ranges split over workgroups, windows of all positions."""
    for lens, new in (([1500], [700]), ([2500], [9]), ([900, 30, 400], [900, 30, 5])):
        pool = Pool(lens, hkv, d, 16, cuda_device, seed=lens[0])
        q = pool.queries(sum(new), heads)
        for f in (dict(softcap=30.0), dict(slopes=slopes_of(heads, cuda_device)), dict(window=300),
                  dict(window=1, softcap=3.0), dict(starts=documents(lens, new, 100)),
                  dict(ends=prefixes(lens, new, [n // 2 for n in lens]), window=200)):
            check_prefill(pool, q, new, d ** -0.5, **f)


@pytest.mark.parametrize("heads,hkv,d", [(14, 2, 64), (8, 2, 128), (4, 2, 32)])
def test_bias_over_many_tiles(cuda_device, heads, hkv, d):
    """Biases that raise or lower the scores from tile to tile, over split and whole key ranges:
    steep and flat, of both signs, none; with ends before, at and behind the position."""
    for lens, new in (([1500, 90], [260, 90]), ([2500], [9])):
        pool = Pool(lens, hkv, d, 16, cuda_device, seed=7)
        q = pool.queries(sum(new), heads)
        slopes = slopes_of(heads, cuda_device)
        slopes[1], slopes[2], slopes[3] = 3.0, -0.25, 0.0
        behind = prefixes(lens, new, [n - 3 for n in lens])
        before = np.concatenate([np.minimum(np.arange(n - k, n) + 1, n // 2) for n, k in zip(lens, new)])
        for f in (dict(), dict(ends=behind), dict(ends=before), dict(softcap=10.0),
                  dict(ends=behind, softcap=10.0), dict(window=600), dict(window=700, softcap=4.0),
                  dict(starts=documents(lens, new, 400))):
            check_prefill(pool, q, new, d ** -0.5, slopes=slopes, **f)


def test_many_sequences(cuda_device):
    """Ragged batches whose workgroups are numbered over the blocks that exist; more than 256."""
    rng = np.random.default_rng(3)
    for count in (60, 300):
        lens = rng.integers(1, 200, count).tolist()
        new = [int(rng.integers(0, n + 1)) for n in lens]
        new[0] = lens[0]
        pool = Pool(lens, 2, 64, 16, cuda_device)
        q = pool.queries(sum(new), 14)
        check_prefill(pool, q, new, 0.125, softcap=7.0, window=40, starts=documents(lens, new, 30),
                      pick=range(0, count, count // 12))


def test_rows_that_see_nothing(cuda_device):
    lens, new = [100, 300, 20, 0], [100, 200, 40, 3]  # the third and last have rows before position 0
    pool = Pool(lens, 2, 64, 16, cuda_device)
    q = pool.queries(sum(new), 14)
    pos = np.concatenate([np.arange(n - k, n) for n, k in zip(lens, new)])
    starts, ends = np.zeros_like(pos), pos + 1
    ends[3:70] = 0          # whole tiles of such rows
    starts[150:160] = 5000
    ends[200:210] = starts[200:210] = 40
    ends[220] = -3
    ends[230] = 2 ** 31 - 1
    starts[240] = -2 ** 31
    out = check_prefill(pool, q, new, 0.125, starts=starts, ends=ends, softcap=6.0)
    empty = (np.maximum(starts, 0) >= np.minimum(ends, np.repeat(lens, new))) | (pos < 0)
    assert empty.sum() > 80 and (out[torch.from_numpy(empty).to(cuda_device)] == 0).all()
    ends[:] = 0
    assert (check_prefill(pool, q, new, 0.125, ends=ends) == 0).all()


@pytest.mark.parametrize("d,heads,hkv", [(64, 14, 2), (128, 8, 2), (256, 4, 1)])
def test_unseen_values_never_reach_a_row(cuda_device, d, heads, hkv):
    """NaN and infinities in keys that some rows see and others do not."""
    lens, new = [500, 260], [300, 260]
    pool = Pool(lens, hkv, d, 16, cuda_device)
    q = pool.queries(sum(new), heads)
    slopes = slopes_of(heads, cuda_device)
    starts = documents(lens, new, 60)
    want = check_prefill(pool, q, new, d ** -0.5, starts=starts, slopes=slopes, window=90)
    loc = pool.ints([0, 300, 560])
    pos = np.concatenate([np.arange(200, 500), np.arange(260)])
    seq = np.repeat([0, 1], new)
    first = np.maximum(np.maximum(starts, pos - 89), 0)
    for b, key, value in ((0, 100, float("nan")), (0, 250, float("inf")), (1, 77, float("nan")),
                          (1, 259, -float("inf")), (0, 499, float("nan"))):
        for target in ("v", "k"):
            kv = {"k": pool.k.clone(), "v": pool.v.clone()}
            kv[target][pool.table[b, key // 16], key % 16] = value
            got = paged_attention_prefill_scored(q, kv["k"], kv["v"], pool.tables, pool.seq_lens, loc, 300,
                                                 d ** -0.5, 0.0, slopes, 90, pool.ints(starts))
            sees = torch.from_numpy((seq == b) & (first <= key) & (key <= pos)).to(cuda_device)
            # (Where the wavefront raises its maxima depends on all its columns: to rounding.)
            assert torch.isfinite(got[~sees]).all()
            assert (got[~sees].float() - want[~sees].float()).abs().max() < 4e-3
            if target == "v" and sees.any():
                assert not torch.isfinite(got[sees]).any()


def test_blocks_before_a_window_hold_anything(cuda_device):
    lens, new = [900, 1400], [40, 300]
    pool = Pool(lens, 2, 64, 16, cuda_device)
    q = pool.queries(sum(new), 14)
    want = check_prefill(pool, q, new, 0.125, window=64, softcap=8.0)
    table = pool.table.copy()
    k, v = pool.k.clone(), pool.v.clone()
    for b, (n, m) in enumerate(zip(lens, new)):
        gone = (n - m - 63) // 16
        k[table[b, :gone]] = float("nan")
        v[table[b, :gone]] = float("nan")
        table[b, :gone] = [(-1, 2 ** 31 - 1, 0)[j % 3] for j in range(gone)]
    got = paged_attention_prefill_scored(q, k, v, torch.from_numpy(table).to(cuda_device), pool.seq_lens,
                                         pool.ints([0, 40, 340]), 300, 0.125, 8.0, None, 64)
    assert torch.equal(got, want)


def test_plain_scores_match_the_plain_kernel(cuda_device):
    pool = Pool([500, 1000], 2, 64, 16, cuda_device)
    q = pool.queries(700, 14)
    args = (q, pool.k, pool.v, pool.tables, pool.seq_lens, pool.ints([0, 200, 700]), 500, 0.125)
    assert (paged_attention_prefill_scored(*args).float() - paged_attention_prefill(*args).float()).abs().max() < 2e-3


def test_rows_of_no_sequence_are_left_alone(cuda_device):
    pool = Pool([50, 60], 2, 64, 16, cuda_device)
    q = pool.queries(100, 14)
    lib = _native.load()
    out = torch.full_like(q, 7.0)
    loc = pool.ints([5, 35, 80])
    st = _native.strides_of
    nbytes = lib.pa_prefill_attention_scored_workspace_bytes(2, 14, 2, 64, 16, pool.tables.shape[1], 45, 0, 0)
    ws = torch.zeros(max(nbytes, 16), dtype=torch.uint8, device=cuda_device)
    status = lib.pa_prefill_attention_scored_f16(
        q.data_ptr(), st(q), pool.k.data_ptr(), st(pool.k), pool.v.data_ptr(), st(pool.v),
        pool.tables.data_ptr(), st(pool.tables), pool.seq_lens.data_ptr(), loc.data_ptr(), 45,
        out.data_ptr(), st(out), 2, 100, 14, 2, 64, 16, pool.blocks, pool.tables.shape[1], 0.125, 9.0,
        None, 1, 0, None, None, ws.data_ptr(), nbytes, _native.stream_handle(q.device))
    _native.check(status, "pa_prefill_attention_scored_f16")
    assert (out[:5] == 7).all() and (out[80:] == 7).all()
    want = check_prefill(pool, q[5:80].contiguous(), [30, 45], 0.125, softcap=9.0)
    assert torch.equal(out[5:80], want)


def test_strides(cuda_device):
    pool = Pool([90, 300], 2, 64, 16, cuda_device)
    new = [50, 200]
    q = pool.queries(250, 14)
    want = check_prefill(pool, q, new, 0.125, softcap=9.0)
    merged = torch.stack([pool.k, pool.v], dim=1)
    wide = torch.zeros(250, 14, 72, dtype=torch.float16, device=cuda_device)
    wide[..., :64] = q
    for qq, k, v in ((q, merged[:, 0], merged[:, 1]), (wide[..., :64], pool.k, pool.v),
                     (q.transpose(0, 1).contiguous().transpose(0, 1), pool.k, pool.v)):
        got = paged_attention_prefill_scored(qq, k, v, pool.tables, pool.seq_lens, pool.ints([0, 50, 250]), 200,
                                             0.125, 9.0)
        assert torch.equal(got, want)


def test_captured(cuda_device):
    with torch.inference_mode():
        pool = Pool([3000, 500], 2, 64, 16, cuda_device)
        q = pool.queries(60, 14)
        args = (pool.k, pool.v, pool.tables, pool.seq_lens, pool.ints([0, 50, 60]), 50, 0.125, 12.0,
                slopes_of(14, cuda_device), 2000)
        paged_attention_prefill_scored(q, *args)
        torch.cuda.synchronize()
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = paged_attention_prefill_scored(q, *args)
            graphs.append((graph, out))
        for i in range(3):
            q.copy_(pool.queries(60, 14, seed=40 + i))
            want = paged_attention_prefill_scored(q, *args)
            for graph, _ in graphs:
                graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(out, want) for _, out in graphs)


def test_nothing_and_refusals(cuda_device):
    pool = Pool([20, 5], 2, 64, 16, cuda_device)
    q = pool.queries(8, 14)
    loc = pool.ints([0, 5, 8])
    rows = torch.zeros(8, dtype=torch.int32, device=cuda_device)

    def call(q=q, loc=loc, most=5, scale=0.125, softcap=0.0, slopes=None, window=0, starts=None, ends=None):
        return paged_attention_prefill_scored(q, pool.k, pool.v, pool.tables, pool.seq_lens, loc, most, scale,
                                              softcap, slopes, window, starts, ends)

    assert call(q=q[:0]).shape == (0, 14, 64)
    for bad in (dict(q=q.float()), dict(q=q[:, :13]), dict(loc=loc[:2]), dict(loc=loc.long()), dict(most=-1),
                dict(window=-1), dict(starts=rows[:5]), dict(ends=rows.long()), dict(ends=rows.cpu()),
                dict(slopes=slopes_of(2, cuda_device))):
        with pytest.raises(AssertionError):
            call(**bad)
    for bad, message in ((dict(scale=-1.0), "scale"), (dict(softcap=float("nan")), "softcap")):
        with pytest.raises(_native.NativeLibraryError, match=message):
            call(**bad)
