"""Sampling's and the block copies' entry points check their arguments before any launch (no GPU)."""
from __future__ import annotations

import pytest
import torch

from engine.kernels import _native
from engine.kernels.cache_blocks import fork_block_table, paged_copy_blocks
from engine.kernels.sampling import sample_tokens, sampling_probs
from engine.memory.block_allocator import BlockAllocator, BlockTable

S = _native.i64_array
P = _native.pointer_array


def _tokens(lib, logits=16, dtype=0, strides=S([100, 0, 1]), u=16, ustr=S([1, 0]), out=16, seqs=2,
            rows=1, vocab=100, ws=16, nbytes=1 << 30):
    return lib.pa_sample_tokens(logits, dtype, strides, u, ustr, None, 1.0, None, 0, None, 1.0, None,
                                0.0, out, seqs, rows, vocab, ws, nbytes, None)


def _probs(lib, logits=16, dtype=0, strides=S([100, 0, 1]), out=16, seqs=2, rows=1, vocab=100, ws=16,
           nbytes=1 << 30):
    return lib.pa_sampling_probs(logits, dtype, strides, None, 1.0, None, 0, None, 1.0, None, 0.0, out,
                                 seqs, rows, vocab, ws, nbytes, None)


@pytest.mark.parametrize("call", [_tokens, _probs])
def test_sampling_argument_errors(call):
    lib = _native.load()
    for bad in (dict(logits=0), dict(out=0), dict(dtype=3), dict(dtype=-1), dict(seqs=-1), dict(rows=-1),
                dict(vocab=0), dict(strides=S([100, 0, 2])), dict(logits=17), dict(logits=18, dtype=2)):
        assert call(lib, **bad) == _native.PA_ERR_ARG, bad
        assert lib.pa_last_error()
    for bad in (dict(seqs=16385), dict(seqs=2 ** 31 - 1, rows=2 ** 31 - 1), dict(vocab=2 ** 19 + 1)):
        assert call(lib, **bad) == _native.PA_ERR_UNSUPPORTED, bad
        assert b"at most" in lib.pa_last_error()
    for bad in (dict(ws=0), dict(nbytes=65536)):
        assert call(lib, **bad) == _native.PA_ERR_WORKSPACE, bad
    for nothing in (dict(seqs=0), dict(rows=0)):
        assert call(lib, logits=0, ws=0, **nothing) == _native.PA_OK
    if call is _tokens:
        assert call(lib, u=0) == _native.PA_ERR_ARG and call(lib, ustr=None) == _native.PA_ERR_ARG


def test_sampling_workspace():
    lib = _native.load()
    assert lib.pa_sample_workspace_bytes(0, 1, 100) == 0
    assert lib.pa_sample_workspace_bytes(1, 1, 2 ** 19 + 1) == 0
    assert lib.pa_sample_workspace_bytes(2 ** 31 - 1, 2 ** 31 - 1, 100) == 0
    one = lib.pa_sample_workspace_bytes(1, 1, 151936)
    # Counters; then for a row its mode, the maxima of its 1187 cells of 128 logits, 16 bytes for
    # each of its 149 pieces of 1024, and 2048 words in which workgroups share a long list.
    assert 65536 < one < 65536 + 16384 + 2048 * 8
    twelve = lib.pa_sample_workspace_bytes(4, 3, 151936)
    assert 65536 + 12 * (one - 65536 - 1024) <= twelve <= 65536 + 12 * (one - 65536)
    assert twelve == lib.pa_sample_workspace_bytes(12, 1, 151936)


def test_copy_argument_errors():
    lib = _native.load()

    def call(tensors=P([4096, 8192]), strides=S([64, 64]), sizes=S([64, 64]), n=2, src=16, dst=16,
             pairs=3, blocks=9):
        return lib.pa_copy_blocks(tensors, strides, sizes, n, src, 1, dst, 1, pairs, blocks, None)

    for bad in (dict(n=-1), dict(pairs=-1), dict(blocks=-1), dict(src=0), dict(dst=0),
                dict(tensors=P([4096, 0])), dict(sizes=S([64, -1])), dict(strides=S([64, 63])),
                dict(tensors=None), dict(strides=None), dict(sizes=None)):
        assert call(**bad) == _native.PA_ERR_ARG, bad
    big = S([2 ** 31, 2 ** 31])
    assert call(sizes=big, strides=big) == _native.PA_ERR_UNSUPPORTED
    big = S([2 ** 30, 2 ** 30])
    assert call(sizes=big, strides=big, pairs=2 ** 31 - 1) == _native.PA_ERR_UNSUPPORTED
    for nothing in (dict(n=0), dict(pairs=0), dict(blocks=0)):
        assert call(tensors=None, src=0, **nothing) == _native.PA_OK


def test_python_calls_need_the_gpu():
    z, one = torch.zeros(2, 10), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: sample_tokens(z, torch.zeros(2)), lambda: sampling_probs(z),
                 lambda: paged_copy_blocks([torch.zeros(4, 8)], one, one)):
        with pytest.raises(AssertionError):
            call()


def test_fork_without_a_partial_block():
    """Full blocks are shared by counts alone: no tensor is touched."""
    alloc = BlockAllocator(8)
    table = BlockTable(seq_id=0, block_size=4, physical_block_ids=[alloc.allocate() for _ in range(2)],
                       num_tokens=8)
    copies = fork_block_table(table, alloc, [], 2)
    assert [t.physical_block_ids for t in copies] == [table.physical_block_ids] * 2
    assert [alloc.ref_counts[b] for b in table.physical_block_ids] == [3, 3]
    copies[0].physical_block_ids.append(99)
    assert 99 not in table.physical_block_ids + copies[1].physical_block_ids
    assert fork_block_table(BlockTable(seq_id=1, block_size=4), alloc, [], 1)[0].num_tokens == 0
    with pytest.raises(AssertionError):
        fork_block_table(BlockTable(seq_id=1, block_size=4, num_tokens=3), alloc, [], 1)


POOL = S([2048, 128, 64, 1])


def _decode(lib, q=16, k=16, out=16, kstr=POOL, qstr=S([896, 64, 1]), hq=14, hkv=2, d=64, bs=16, blocks=10,
            width=4, seqs=2, scale=0.125, softcap=0.0, window=0, ws=0, nbytes=0):
    return lib.pa_decode_scored_f16(q, qstr, k, kstr, 16, POOL, 16, S([4, 1]), 16, out, S([896, 64, 1]), seqs,
                                    hq, hkv, d, bs, blocks, width, scale, softcap, None, 1, window, None, ws,
                                    nbytes, None)


def _prefill(lib, q=16, k=16, out=16, kstr=POOL, qstr=S([896, 64, 1]), hq=14, hkv=2, d=64, bs=16, blocks=10,
             width=4, seqs=2, scale=0.125, softcap=0.0, window=0, ws=0, nbytes=0):
    return lib.pa_prefill_attention_scored_f16(q, qstr, k, kstr, 16, POOL, 16, S([4, 1]), 16, 16, 9, out,
                                               S([896, 64, 1]), seqs, 9, hq, hkv, d, bs, blocks, width, scale,
                                               softcap, None, 1, window, None, None, ws, nbytes, None)


@pytest.mark.parametrize("call", [_decode, _prefill])
def test_scored_attention_argument_errors(call):
    lib = _native.load()
    nan, inf = float("nan"), float("inf")
    for bad in (dict(q=0), dict(out=0), dict(k=8), dict(hq=15), dict(hkv=0), dict(bs=0), dict(blocks=0),
                dict(width=0), dict(seqs=-1), dict(kstr=S([2048, 128, 60, 1])), dict(kstr=S([2048, 128, 64, 2])),
                dict(qstr=S([900, 64, 1])), dict(qstr=S([896, 64, 2])), dict(scale=0.0), dict(scale=-1.0),
                dict(scale=nan), dict(scale=inf), dict(softcap=-1.0), dict(softcap=nan), dict(softcap=inf),
                dict(window=-1)):
        assert call(lib, **bad) == _native.PA_ERR_ARG, bad
        assert lib.pa_last_error()
    for bad in (dict(hq=34), dict(d=48, qstr=S([896, 64, 1])), dict(width=2 ** 28)):
        assert call(lib, **bad) == _native.PA_ERR_UNSUPPORTED, bad
    assert call(lib, q=0, seqs=0) == _native.PA_OK


def test_scored_attention_workspace():
    lib = _native.load()
    # Windows and short tables need none; what a window bounds needs no more than the table.
    decode = lib.pa_decode_scored_workspace_bytes
    assert decode(4, 14, 2, 64, 16, 32, 0) == 0 and decode(4, 14, 2, 64, 16, 2048, 512) == 0
    assert decode(4, 14, 2, 64, 16, 2048, 0) >= decode(4, 14, 2, 64, 16, 2048, 4096) > 65536
    assert decode(4, 34, 2, 64, 16, 2048, 0) == 0
    prefill = lib.pa_prefill_attention_scored_workspace_bytes
    assert prefill(1, 14, 2, 64, 16, 512, 64, 0, 0) == lib.pa_prefill_attention_workspace_bytes(
        1, 14, 2, 64, 16, 512, 64)
    assert prefill(1, 14, 2, 64, 16, 512, 64, 100, 0) < prefill(1, 14, 2, 64, 16, 512, 64, 100, 1)


def test_refused_forks_leave_the_counts():
    """Copies that are refused (here: off the GPU, no tensors, blocks run out) cost no block."""
    import torch
    from engine.kernels.cache_blocks import fork_block_table
    from engine.memory.block_allocator import BlockAllocator, BlockTable

    alloc = BlockAllocator(5)
    table = BlockTable(seq_id=0, block_size=4)
    table.physical_block_ids = [alloc.allocate() for _ in range(2)]
    table.num_tokens = 7
    before = dict(alloc.ref_counts)
    caches = [torch.zeros(5, 4, 2, 8, dtype=torch.float16)]
    for args in ((caches, 2), ([], 1), (caches, 4)):
        with pytest.raises(Exception):
            fork_block_table(table, alloc, *args)
        assert {k: v for k, v in alloc.ref_counts.items() if v} == before
    assert len([alloc.allocate() for _ in range(3)]) == 3
    # Full blocks alone are shared without a copy.
    table.num_tokens = 8
    forks = fork_block_table(table, alloc, caches, 2)
    assert [f.physical_block_ids for f in forks] == [table.physical_block_ids] * 2
    assert all(alloc.ref_counts[b] == 3 for b in table.physical_block_ids)
