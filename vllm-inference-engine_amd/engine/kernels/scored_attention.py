"""Paged attention with capped, biased and masked scores.

No counterpart in the reference, whose kernels compute plain causal scores
(engine/kernels/paged_attention.py:508-698). For a query row at position p of head h and
key j of its sequence, with x = scale * q.k_j:

  s = softcap * tanh(x / softcap)   (softcap 0: x itself; both at most 2^127)
  s = s - alibi_slopes[h] * |p - j| (None: no bias)

and the output is softmax(s) v over the keys that the row sees. window W > 0: none before
p - W + 1. A row that sees no key is zeros. What lies in keys that a row does not see never
reaches it, NaN included: the blocks that a window has left behind may be freed and hold
anything. A NaN or an infinity in a V row makes the rows that see it NaN or infinite (all of
head_dim or a part).

Pools, tables, lengths and rows are those of paged_attention_decode_batched and
paged_attention_prefill: fp16, head_dim 32, 64, 128 or 256, query groups of up to 16.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _native
from .paged_attention import _on_device, _q_ready

__all__ = [
    "paged_attention_decode_scored",
    "paged_attention_prefill_scored",
]

# Bytes of the arrival counters at the head of the workspaces (16384 ints).
_COUNTER_BYTES = 65536


def _check(q, k_cache, v_cache, block_tables, seq_lens, alibi_slopes, window):
    """What both calls ask; (q, seq_lens, slopes, window)."""
    assert q.is_cuda and k_cache.is_cuda and v_cache.is_cuda
    assert block_tables.is_cuda and seq_lens.is_cuda
    _native.same_device(q, k_cache, v_cache, block_tables, seq_lens)
    assert q.dtype == torch.float16 and k_cache.dtype == torch.float16 and v_cache.dtype == torch.float16
    assert block_tables.dtype == torch.int32 and seq_lens.dtype == torch.int32
    assert k_cache.dim() == 4 and v_cache.shape == k_cache.shape, (
        "k_cache and v_cache must have the same [num_blocks, block_size, num_kv_heads, head_dim]")
    num_kv_heads, head_dim = k_cache.shape[2:]
    assert q.dim() == 3 and q.shape[2] == head_dim, (
        f"queries must be [tokens, num_q_heads, {head_dim}], got {tuple(q.shape)}")
    assert num_kv_heads > 0 and q.shape[1] % num_kv_heads == 0, (
        f"num_q_heads ({q.shape[1]}) must be divisible by num_kv_heads ({num_kv_heads})")
    assert block_tables.dim() == 2 and seq_lens.dim() == 1
    assert block_tables.shape[0] == seq_lens.shape[0]
    if alibi_slopes is not None:
        assert alibi_slopes.is_cuda and alibi_slopes.dtype == torch.float32
        _native.same_device(alibi_slopes, q)
        assert alibi_slopes.shape == (q.shape[1],), (
            f"alibi_slopes must have one entry per query head ({q.shape[1]}), got "
            f"{tuple(alibi_slopes.shape)}")
    assert window >= 0, f"window must be 0 (none) or positive, got {window}"
    if window >= block_tables.shape[1] * k_cache.shape[1]:
        window = 0  # all that the table can hold
    return _q_ready(q), seq_lens.contiguous(), alibi_slopes, window


def _keys(name: str, x: Optional[torch.Tensor], n: int, like: torch.Tensor):
    if x is None:
        return None
    assert x.is_cuda and x.dtype == torch.int32, f"{name} must be int32 on the GPU"
    _native.same_device(x, like)
    assert x.shape == (n,), f"{name} must have {n} entries, got {tuple(x.shape)}"
    return x.contiguous()


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def paged_attention_decode_scored(
    q: torch.Tensor,             # [num_seqs, num_q_heads, head_dim] fp16
    k_cache: torch.Tensor,       # [num_blocks, block_size, num_kv_heads, head_dim] fp16
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,  # [num_seqs, max_blocks_per_seq] int32
    seq_lens: torch.Tensor,      # [num_seqs] int32
    scale: float,
    softcap: float = 0.0,
    alibi_slopes: Optional[torch.Tensor] = None,  # [num_q_heads] fp32
    window: int = 0,
    key_starts: Optional[torch.Tensor] = None,    # [num_seqs] int32: first key seen
) -> torch.Tensor:
    """Batched GQA decode attention with the module's scores, one query token per sequence.

    The token stands at position p = seq_lens[b] - 1 and sees keys max(key_starts[b],
    p - window + 1, 0) .. p. Lengths, tables and block ids out of range are treated as in
    paged_attention_decode_batched. One launch; long contexts are split over workgroups that
    merge in it, through a per-stream scratch buffer (the graph's own while one is captured).
    Repeated calls return the same bits.
    """
    window = int(window)
    out = _native.direct_counted("decode_scored", _native.WS_DECODE_SCORED, q, k_cache, v_cache,
                                 block_tables, seq_lens, float(scale), float(softcap), alibi_slopes,
                                 window, key_starts)
    if out is not None:
        return out
    q, seq_lens, slopes, window = _check(q, k_cache, v_cache, block_tables, seq_lens, alibi_slopes,
                                         window)
    num_seqs, num_q_heads, head_dim = q.shape
    assert seq_lens.shape[0] == num_seqs
    key_starts = _keys("key_starts", key_starts, num_seqs, q)
    num_blocks, block_size, num_kv_heads, _ = k_cache.shape
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if num_seqs == 0 or num_q_heads == 0:
        return out
    lib = _native.load()
    dev = q.device
    st = _native.strides_of
    max_blocks = block_tables.shape[1]
    stream = _native.stream_handle(dev)
    with _on_device(dev):
        nbytes = lib.pa_decode_scored_workspace_bytes(num_seqs, num_q_heads, num_kv_heads, head_dim,
                                                      block_size, max_blocks, window)
        ws, _own = _native.counted_workspace(nbytes, _COUNTER_BYTES, dev, stream,
                                             _native.WS_DECODE_SCORED)
        status = lib.pa_decode_scored_f16(
            q.data_ptr(), st(q), k_cache.data_ptr(), st(k_cache), v_cache.data_ptr(), st(v_cache),
            block_tables.data_ptr(), st(block_tables), seq_lens.data_ptr(), out.data_ptr(), st(out),
            num_seqs, num_q_heads, num_kv_heads, head_dim, block_size, num_blocks, max_blocks,
            float(scale), float(softcap), _ptr(slopes), 1 if slopes is None else slopes.stride(0),
            window, _ptr(key_starts), ws, nbytes, stream)
    _native.check(status, "pa_decode_scored_f16")
    return out


def paged_attention_prefill_scored(
    q: torch.Tensor,                # [num_tokens, num_q_heads, head_dim] fp16
    k_cache: torch.Tensor,          # [num_blocks, block_size, num_kv_heads, head_dim] fp16
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,     # [num_seqs, max_blocks_per_seq] int32
    seq_lens: torch.Tensor,         # [num_seqs] int32: context length after the new tokens
    query_start_loc: torch.Tensor,  # [num_seqs + 1] int32: first q row of each sequence
    max_query_len: int,
    scale: float,
    softcap: float = 0.0,
    alibi_slopes: Optional[torch.Tensor] = None,  # [num_q_heads] fp32
    window: int = 0,
    key_starts: Optional[torch.Tensor] = None,    # [num_tokens] int32: first key of each row
    key_ends: Optional[torch.Tensor] = None,      # [num_tokens] int32: end of each row's keys
) -> torch.Tensor:
    """Attention of each sequence's new tokens over its paged context with the module's scores.

    Rows and positions as in paged_attention_prefill. The row at position p sees keys from
    max(key_starts, p - window + 1, 0) on and before min(key_ends, seq_lens[b]); without
    key_ends those up to its own position. Packed documents: key_starts = the first key of the
    row's document. A prefix that is seen as a whole: key_ends = max(p + 1, its length). scale
    must be positive; rows of q that belong to no sequence, or lie past max_query_len, are not
    written.
    """
    window, max_query_len = int(window), int(max_query_len)
    out = _native.direct_counted("prefill_scored", _native.WS_PREFILL, q, k_cache, v_cache,
                                 block_tables, seq_lens, query_start_loc, max_query_len,
                                 float(scale), float(softcap), alibi_slopes, window, key_starts,
                                 key_ends)
    if out is not None:
        return out
    q, seq_lens, slopes, window = _check(q, k_cache, v_cache, block_tables, seq_lens, alibi_slopes,
                                         window)
    num_tokens, num_q_heads, head_dim = q.shape
    num_seqs = seq_lens.shape[0]
    assert query_start_loc.is_cuda and query_start_loc.dtype == torch.int32
    _native.same_device(query_start_loc, q)
    assert query_start_loc.dim() == 1 and query_start_loc.shape[0] == num_seqs + 1
    query_start_loc = query_start_loc.contiguous()
    key_starts = _keys("key_starts", key_starts, num_tokens, q)
    key_ends = _keys("key_ends", key_ends, num_tokens, q)
    assert 0 <= max_query_len < 2 ** 31
    num_blocks, block_size, num_kv_heads, _ = k_cache.shape
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if num_seqs == 0 or num_tokens == 0 or num_q_heads == 0 or max_query_len == 0:
        return out
    lib = _native.load()
    dev = q.device
    st = _native.strides_of
    max_blocks = block_tables.shape[1]
    stream = _native.stream_handle(dev)
    with _on_device(dev):
        nbytes = lib.pa_prefill_attention_scored_workspace_bytes(
            num_seqs, num_q_heads, num_kv_heads, head_dim, block_size, max_blocks, max_query_len,
            window, key_ends is not None)
        ws, _own = _native.counted_workspace(nbytes, _COUNTER_BYTES, dev, stream, _native.WS_PREFILL)
        status = lib.pa_prefill_attention_scored_f16(
            q.data_ptr(), st(q), k_cache.data_ptr(), st(k_cache), v_cache.data_ptr(), st(v_cache),
            block_tables.data_ptr(), st(block_tables), seq_lens.data_ptr(),
            query_start_loc.data_ptr(), max_query_len, out.data_ptr(), st(out), num_seqs, num_tokens,
            num_q_heads, num_kv_heads, head_dim, block_size, num_blocks, max_blocks, float(scale),
            float(softcap), _ptr(slopes), 1 if slopes is None else slopes.stride(0), window,
            _ptr(key_starts), _ptr(key_ends), ws, nbytes, stream)
    _native.check(status, "pa_prefill_attention_scored_f16")
    return out
