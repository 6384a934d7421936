"""Decode attention with capped, biased and windowed scores against the 64-bit oracle (needs an MI355X)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from _scored import Pool, check_decode, slopes_of
from engine.kernels import _native
from engine.kernels.paged_attention import paged_attention_decode_batched
from engine.kernels.scored_attention import paged_attention_decode_scored

pytestmark = pytest.mark.gpu

FORMS = [dict(), dict(softcap=20.0), dict(bias=True), dict(window=100), dict(softcap=5.0, bias=True, window=33)]


def form(pool, heads, bias=False, **rest):
    return dict(rest, slopes=slopes_of(heads, pool.device) if bias else None)


@pytest.mark.parametrize("heads,hkv,d", [(14, 2, 64), (32, 8, 128), (16, 16, 64), (4, 2, 32), (16, 2, 256),
                                         (16, 1, 64), (3, 3, 128), (5, 1, 128), (12, 1, 256)])
@pytest.mark.parametrize("bs", [16, 32, 8, 5])
def test_shapes(cuda_device, heads, hkv, d, bs):
    pool = Pool([1, 17, 32, 33, 300, 511, 64], hkv, d, bs, cuda_device, seed=d + bs)
    q = pool.queries(7, heads)
    for f in FORMS:
        check_decode(pool, q, d ** -0.5, **form(pool, heads, **f))


@pytest.mark.parametrize("lens", [[9000], [5000, 1, 0, 3100], [2500] * 40, list(range(1, 3000, 10))])
@pytest.mark.parametrize("heads,hkv,d,bs", [(14, 2, 64, 16), (8, 2, 128, 16), (4, 2, 256, 16), (8, 8, 64, 8),
                                            (2, 1, 32, 32)])
def test_long_contexts(cuda_device, lens, heads, hkv, d, bs):
    """Contexts cut into ranges of workgroups; more than 256 sequences."""
    pool = Pool(lens, hkv, d, bs, cuda_device, seed=len(lens))
    q = pool.queries(len(lens), heads)
    pick = range(0, len(lens), max(1, len(lens) // 6))
    for f in (dict(softcap=30.0), dict(bias=True), dict(window=2100), dict(window=1500, softcap=30.0)):
        check_decode(pool, q, d ** -0.5, pick=pick, **form(pool, heads, **f))


def test_first_keys_and_rows_that_see_nothing(cuda_device):
    lens = [0, 1, 40, 40, 40, 40, 3000, 3000, 3000, -5]
    pool = Pool(lens, 2, 64, 16, cuda_device)
    q = pool.queries(len(lens), 14)
    for starts in ([0, 0, 39, 40, 41, 31, 2999, 3000, 5, 0], [-7, 5, 2 ** 31 - 1, 33, 32, 1, 2000, 999, 1, 9]):
        for window in (0, 7, 1200):
            out = check_decode(pool, q, 0.125, softcap=10.0, starts=starts, window=window)
            for b, n in enumerate(lens):
                if starts[b] >= n:
                    assert (out[b] == 0).all()


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 64, 4095, 4096, 4097, 10 ** 9])
def test_windows(cuda_device, window):
    pool = Pool([4096, 50, 4095], 2, 64, 16, cuda_device)
    check_decode(pool, pool.queries(3, 14), 0.125, window=window, slopes=slopes_of(14, cuda_device))


@pytest.mark.parametrize("bs", [16, 8])
def test_what_a_window_left_behind_never_reaches_a_result(cuda_device, bs):
    """NaN, infinities and ids out of the pool before the window and behind the last token."""
    lens = [400, 37, 3000]
    pool = Pool(lens, 2, 64, bs, cuda_device)
    q = pool.queries(3, 14)
    window = 50
    want = check_decode(pool, q, 0.125, window=window, softcap=8.0)
    kv = [x.clone() for x in (pool.k, pool.v)]
    table = pool.table.copy()
    for b, n in enumerate(lens):
        for j in list(range(0, max(0, n - window))) + list(range(n, -(-n // bs) * bs)):
            for x in kv:
                x[table[b, j // bs], j % bs] = (float("nan"), float("inf"), -float("inf"))[j % 3]
        gone = max(0, n - window) // bs  # whole blocks before the window
        table[b, :gone] = [(-1, 2 ** 31 - 1, pool.blocks)[j % 3] for j in range(gone)]
    got = paged_attention_decode_scored(q, *kv, torch.from_numpy(table).to(cuda_device), pool.seq_lens,
                                        0.125, 8.0, None, window)
    assert torch.equal(got, want)
    # A NaN that is seen shows, in its head's rows and in no other.
    kv[1][pool.table[1, 36 // bs], 36 % bs, 1, 5] = float("nan")
    got = paged_attention_decode_scored(q, *kv, pool.tables, pool.seq_lens, 0.125, 8.0, None, window)
    assert torch.isnan(got[1, 7:, 5]).all() and torch.equal(got[1, :7], want[1, :7])
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])


def test_large_scores(cuda_device):
    """Scores of tens of thousands, capped and not; a cap far above and far below them."""
    pool = Pool([700, 3], 2, 128, 16, cuda_device)
    q = pool.queries(2, 8, spread=300.0)
    for softcap in (0.5, 50.0, 1e6):
        out = check_decode(pool, q, 1.0, softcap=softcap)
        assert torch.isfinite(out).all()
    assert torch.isfinite(check_decode(pool, q, 1.0)).all()


def test_plain_scores_match_the_plain_kernel(cuda_device):
    pool = Pool([500, 3000, 20], 2, 64, 16, cuda_device)
    q = pool.queries(3, 14)
    a = paged_attention_decode_scored(q, pool.k, pool.v, pool.tables, pool.seq_lens, 0.125)
    b = paged_attention_decode_batched(q, pool.k, pool.v, pool.tables, pool.seq_lens, 0.125)
    assert (a.float() - b.float()).abs().max() < 2e-3


def test_strides(cuda_device):
    pool = Pool([90, 700], 2, 64, 16, cuda_device)
    q = pool.queries(2, 14)
    want = check_decode(pool, q, 0.125, softcap=9.0)
    merged = torch.stack([pool.k, pool.v], dim=1)  # one tensor of K and V blocks
    heads_first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (pool.k, pool.v)]
    wide = torch.zeros(2, 14, 72, dtype=torch.float16, device=cuda_device)
    wide[..., :64] = q
    odd = torch.zeros(2, 14, 67, dtype=torch.float16, device=cuda_device)
    odd[..., 3:] = q
    tables = pool.tables.t().contiguous().t()
    for other in (dict(k=merged[:, 0], v=merged[:, 1]), dict(k=heads_first[0], v=heads_first[1]),
                  dict(q=wide[..., :64]), dict(q=odd[..., 3:]), dict(tables=tables)):
        got = paged_attention_decode_scored(other.get("q", q), other.get("k", pool.k), other.get("v", pool.v),
                                            other.get("tables", pool.tables), pool.seq_lens, 0.125, 9.0)
        assert torch.equal(got, want)
    slopes = torch.stack([slopes_of(14, cuda_device)] * 2, dim=1)
    assert torch.equal(
        paged_attention_decode_scored(q, pool.k, pool.v, pool.tables, pool.seq_lens, 0.125, 0.0, slopes[:, 0]),
        paged_attention_decode_scored(q, pool.k, pool.v, pool.tables, pool.seq_lens, 0.125, 0.0,
                                      slopes_of(14, cuda_device)))


def test_far_offsets(cuda_device):
    """Blocks past 2^31 elements and bytes of a large pool."""
    blocks = 140000
    k = torch.zeros(blocks, 16, 8, 128, dtype=torch.float16, device=cuda_device)
    v = torch.zeros(blocks, 16, 8, 128, dtype=torch.float16, device=cuda_device)
    ids = torch.tensor([[blocks - 1, 5, blocks // 2 + 7]], dtype=torch.int32, device=cuda_device)
    pool = Pool([45], 8, 128, 16, cuda_device, spare=0)
    for x, y in ((k, pool.k), (v, pool.v)):
        x[ids[0].long()] = y[pool.tables[0].long()]
    q = pool.queries(1, 32)
    want = check_decode(pool, q, 0.1, softcap=5.0)
    got = paged_attention_decode_scored(q, k, v, ids, pool.seq_lens, 0.1, 5.0)
    assert torch.equal(got, want)


def test_captured_repeated_and_on_another_stream(cuda_device):
    with torch.inference_mode():
        pool = Pool([3000, 10, 6000, 2000], 2, 64, 16, cuda_device)
        q = pool.queries(4, 14)
        args = (pool.k, pool.v, pool.tables, pool.seq_lens, 0.125, 12.0, slopes_of(14, cuda_device), 2500)
        want = paged_attention_decode_scored(q, *args)
        for _ in range(3):
            assert torch.equal(paged_attention_decode_scored(q, *args), want)
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = paged_attention_decode_scored(q, *args)
            graphs.append((graph, out))
        side = torch.cuda.Stream()
        for i in range(3):
            q.copy_(pool.queries(4, 14, seed=30 + i))
            want = paged_attention_decode_scored(q, *args)
            for graph, _ in graphs:
                graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(out, want) for _, out in graphs)
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                got = paged_attention_decode_scored(q, *args)
            torch.cuda.current_stream().wait_stream(side)
            assert torch.equal(got, want)


def test_nothing_and_refusals(cuda_device):
    pool = Pool([20, 5], 2, 64, 16, cuda_device)
    q = pool.queries(2, 14)

    def call(q=q, k=pool.k, scale=0.125, softcap=0.0, slopes=None, window=0, starts=None, lens=pool.seq_lens,
             tables=pool.tables):
        return paged_attention_decode_scored(q, k, pool.v, tables, lens, scale, softcap, slopes, window, starts)

    assert call(q=q[:0], lens=pool.seq_lens[:0], tables=pool.tables[:0]).shape == (0, 14, 64)
    for bad in (dict(q=q.float()), dict(q=q[:, :13]), dict(q=q.cpu()), dict(window=-1), dict(k=pool.k[:, :8]),
                dict(slopes=slopes_of(13, cuda_device)), dict(slopes=slopes_of(14, cuda_device).double()),
                dict(starts=torch.zeros(3, dtype=torch.int32, device=cuda_device)),
                dict(starts=torch.zeros(2, device=cuda_device)), dict(lens=pool.seq_lens.long()),
                dict(lens=pool.seq_lens[:1])):
        with pytest.raises(AssertionError):
            call(**bad)
    for bad, message in ((dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
                         (dict(softcap=-1.0), "softcap"), (dict(softcap=float("inf")), "softcap"),
                         (dict(q=pool.queries(2, 34)), "group")):
        with pytest.raises(_native.NativeLibraryError, match=message):
            call(**bad)
