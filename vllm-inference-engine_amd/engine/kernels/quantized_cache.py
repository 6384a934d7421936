"""The paged KV pool in 8 bits: writing it, reading it back, attention over it.

No counterpart in the reference, whose pool is fp16
(engine/memory/block_allocator.py:101). A pool of one layer is four tensors:

  k_cache, v_cache  [num_blocks, block_size, num_kv_heads, head_dim] torch.float8_e4m3fn
  k_scale, v_scale  [num_blocks, num_kv_heads] fp32

A value is code * scale[block, head]. Scales are powers of two from 2^-15 to 2^8,
as paged_kv_write_fp8 leaves them (of a scale between two powers every call takes the
lower one: a pool coded with others has to be coded again): every value is then an
fp16 number, and a block whose scale grows as it fills is coded again without a
second rounding (but for codes that fall below e4m3's normal range). A fresh pool
needs no initial values: a write that begins a block sets its scale. Half the bytes of
the fp16 pool (plus 8 bytes per block and head), for a rounding of at most 2^-4 of each
value, or for values below 2^-6 times their scale of 2^-10 times it (once more where
they are coded again).

Several tokens per sequence are described as for paged_attention_prefill: sequence
b owns rows query_start_loc[b] .. query_start_loc[b + 1] - 1 of a packed row list,
which stand at the last positions of its seq_lens[b] tokens. Every call is
asynchronous on the current stream and reads nothing on the host; block ids outside
the pool and positions outside the table never reach memory.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _native
from .paged_attention import _on_device, _q_ready

__all__ = [
    "paged_kv_write_fp8",
    "paged_kv_read_fp8",
    "paged_attention_decode_fp8",
    "paged_attention_prefill_fp8",
]


def _check_pool(k_cache, v_cache, k_scale, v_scale, block_tables, seq_lens):
    """What every call asks of the pool, the tables and the lengths; (block_tables, seq_lens)."""
    assert k_cache.is_cuda and v_cache.is_cuda and k_scale.is_cuda and v_scale.is_cuda
    assert block_tables.is_cuda and seq_lens.is_cuda
    _native.same_device(k_cache, v_cache, k_scale, v_scale, block_tables, seq_lens)
    assert k_cache.dtype == torch.float8_e4m3fn and v_cache.dtype == torch.float8_e4m3fn, (
        f"the pool holds float8_e4m3fn codes, got {k_cache.dtype} and {v_cache.dtype}")
    assert k_scale.dtype == torch.float32 and v_scale.dtype == torch.float32
    assert block_tables.dtype == torch.int32 and seq_lens.dtype == torch.int32
    assert k_cache.dim() == 4 and v_cache.shape == k_cache.shape, (
        "k_cache and v_cache must have the same [num_blocks, block_size, num_kv_heads, head_dim]")
    scales = (k_cache.shape[0], k_cache.shape[2])
    assert k_scale.shape == scales and v_scale.shape == scales, (
        f"scales must be [num_blocks, num_kv_heads] = {scales}, got {tuple(k_scale.shape)} "
        f"and {tuple(v_scale.shape)}")
    assert block_tables.dim() == 2 and seq_lens.dim() == 1
    assert block_tables.shape[0] == seq_lens.shape[0]
    return block_tables, seq_lens.contiguous()


def _check_starts(query_start_loc: torch.Tensor, like: torch.Tensor, num_seqs: int) -> torch.Tensor:
    assert query_start_loc.is_cuda and query_start_loc.dtype == torch.int32
    _native.same_device(query_start_loc, like)
    assert query_start_loc.dim() == 1 and query_start_loc.shape[0] == num_seqs + 1
    return query_start_loc.contiguous()


def _check_queries(q: torch.Tensor, k_cache: torch.Tensor) -> None:
    assert q.is_cuda and q.dtype == torch.float16
    _native.same_device(q, k_cache)
    assert q.dim() == 3 and q.shape[2] == k_cache.shape[3], (
        f"queries must be [tokens, num_q_heads, {k_cache.shape[3]}], got {tuple(q.shape)}")
    assert k_cache.shape[2] > 0 and q.shape[1] % k_cache.shape[2] == 0, (
        f"num_q_heads ({q.shape[1]}) must be divisible by num_kv_heads ({k_cache.shape[2]})")


def paged_kv_write_fp8(
    key: torch.Tensor,           # [num_tokens, num_kv_heads, head_dim] fp16, any strides
    value: torch.Tensor,         # same
    k_cache: torch.Tensor,       # [num_blocks, block_size, num_kv_heads, head_dim] float8_e4m3fn
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,       # [num_blocks, num_kv_heads] fp32
    v_scale: torch.Tensor,
    block_tables: torch.Tensor,  # [num_seqs, max_blocks_per_seq] int32
    seq_lens: torch.Tensor,      # [num_seqs] int32, the new tokens counted
    query_start_loc: Optional[torch.Tensor] = None,  # [num_seqs + 1] int32
) -> None:
    """Write each sequence's newest K/V rows into its slots as e4m3 codes.

    Without query_start_loc every sequence writes one row (key may then be
    [num_seqs, num_kv_heads, 1, head_dim], as for paged_kv_write) at position
    seq_lens[b] - 1; with it, sequence b writes its n_b rows at positions
    seq_lens[b] - n_b .. seq_lens[b] - 1: a prompt, a chunk of one, or drafted tokens.

    Each touched (block, kv head) gets the smallest power-of-two scale that holds its
    new rows within e4m3's 448, but not less than the present one where earlier rows
    stay in the block; if it grew, those rows are coded again. |x| above 61440 is
    taken as 61440, NaN stays NaN. Rows without a slot (negative positions, blocks
    outside the table or the pool) are skipped, and a call repeated changes nothing.
    Rows of a written block that lie behind the new ones (tokens taken back) keep
    their codes but not their values. No two sequences may write the same block.
    """
    if _native.direct_call("write_fp8", key, value, k_cache, v_cache, k_scale, v_scale,
                           block_tables, seq_lens, query_start_loc):
        return
    block_tables, seq_lens = _check_pool(k_cache, v_cache, k_scale, v_scale, block_tables,
                                         seq_lens)
    num_seqs = seq_lens.shape[0]
    if query_start_loc is None:
        if key.dim() == 4:
            assert key.shape[2] == 1 and value.dim() == 4 and value.shape[2] == 1, (
                f"expected one new token per sequence, got {tuple(key.shape)}")
            key, value = key.squeeze(2), value.squeeze(2)
        assert key.shape[0] == num_seqs, (
            f"{key.shape[0]} rows for {num_seqs} sequences need query_start_loc")
        starts = None
    else:
        query_start_loc = _check_starts(query_start_loc, k_cache, num_seqs)
        starts = query_start_loc.data_ptr()
    _native.same_device(key, value, k_cache)
    assert key.dtype == torch.float16 and value.dtype == torch.float16
    num_blocks, block_size, num_kv_heads, head_dim = k_cache.shape
    assert key.dim() == 3 and key.shape[1:] == (num_kv_heads, head_dim), (
        f"key shape {tuple(key.shape)} does not match the pool ({num_kv_heads}, {head_dim})")
    assert value.shape == key.shape, f"value shape {tuple(value.shape)} != key shape {tuple(key.shape)}"
    num_tokens = key.shape[0]
    if num_tokens == 0 or num_seqs == 0:
        return
    lib = _native.load()
    dev = key.device
    st = _native.strides_of
    with _on_device(dev):
        status = lib.pa_kv_write_fp8(
            key.data_ptr(), st(key), value.data_ptr(), st(value),
            k_cache.data_ptr(), st(k_cache), v_cache.data_ptr(), st(v_cache),
            k_scale.data_ptr(), st(k_scale), v_scale.data_ptr(), st(v_scale),
            block_tables.data_ptr(), st(block_tables), seq_lens.data_ptr(), starts,
            num_seqs, num_tokens, num_kv_heads, head_dim, block_size, num_blocks,
            block_tables.shape[1], _native.stream_handle(dev))
    _native.check(status, "pa_kv_write_fp8")


def paged_kv_read_fp8(
    k_cache: torch.Tensor,          # [num_blocks, block_size, num_kv_heads, head_dim] float8_e4m3fn
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,          # [num_blocks, num_kv_heads] fp32
    v_scale: torch.Tensor,
    block_tables: torch.Tensor,     # [num_seqs, max_blocks_per_seq] int32
    seq_lens: torch.Tensor,         # [num_seqs] int32
    query_start_loc: torch.Tensor,  # [num_seqs + 1] int32: first output row of each sequence
    num_tokens: int,                # output rows
) -> Tuple[torch.Tensor, torch.Tensor]:
    """The sequences' last n_b K/V rows as fp16: (key, value) [num_tokens, num_kv_heads, head_dim].

    The rows paged_kv_write_fp8 writes for the same lengths and starts: with
    n_b = seq_lens[b] the whole contexts, one after the other. Exact (each value is an
    fp16 number). Rows without a slot, and rows of no sequence, are zeros.
    """
    num_tokens = int(num_tokens)
    out = _native.direct_call("read_fp8", k_cache, v_cache, k_scale, v_scale, block_tables,
                              seq_lens, query_start_loc, num_tokens)
    if out is not None:
        return out
    block_tables, seq_lens = _check_pool(k_cache, v_cache, k_scale, v_scale, block_tables,
                                         seq_lens)
    num_seqs = seq_lens.shape[0]
    query_start_loc = _check_starts(query_start_loc, k_cache, num_seqs)
    assert 0 <= num_tokens < 2 ** 31
    num_blocks, block_size, num_kv_heads, head_dim = k_cache.shape
    dev = k_cache.device
    shape = (num_tokens, num_kv_heads, head_dim)
    if num_seqs == 0:
        return (torch.zeros(shape, dtype=torch.float16, device=dev),
                torch.zeros(shape, dtype=torch.float16, device=dev))
    key = torch.empty(shape, dtype=torch.float16, device=dev)
    value = torch.empty_like(key)
    if num_tokens == 0:
        return key, value
    lib = _native.load()
    st = _native.strides_of
    with _on_device(dev):
        status = lib.pa_kv_read_fp8(
            k_cache.data_ptr(), st(k_cache), v_cache.data_ptr(), st(v_cache),
            k_scale.data_ptr(), st(k_scale), v_scale.data_ptr(), st(v_scale),
            block_tables.data_ptr(), st(block_tables), seq_lens.data_ptr(),
            query_start_loc.data_ptr(), key.data_ptr(), st(key), value.data_ptr(), st(value),
            num_seqs, num_tokens, num_kv_heads, head_dim, block_size, num_blocks,
            block_tables.shape[1], _native.stream_handle(dev))
    _native.check(status, "pa_kv_read_fp8")
    return key, value


_ws_sizes: dict = {}
# Bytes of the arrival counters at the head of the attention workspaces (16384 ints).
_COUNTER_BYTES = 65536


def paged_attention_decode_fp8(
    q: torch.Tensor,             # [num_seqs, num_q_heads, head_dim] fp16
    k_cache: torch.Tensor,       # [num_blocks, block_size, num_kv_heads, head_dim] float8_e4m3fn
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,       # [num_blocks, num_kv_heads] fp32
    v_scale: torch.Tensor,
    block_tables: torch.Tensor,  # [num_seqs, max_blocks_per_seq] int32
    seq_lens: torch.Tensor,      # [num_seqs] int32
    scale: float,
) -> torch.Tensor:
    """Batched GQA decode attention over the 8-bit pool: paged_attention_decode_batched on
    K and V rows = code * scale[block, head].

    The same lengths, tables and refusals: head_dim 32, 64, 128 or 256, query groups of up
    to 16, seq_lens 0 gives zeros, lengths past the table are cut to it and block ids
    clamped into the pool. One launch; long contexts are split over workgroups that merge
    in it, through a per-stream scratch buffer (the graph's own while one is captured).
    Repeated calls return the same bits.
    """
    out = _native.direct_counted("decode_fp8", _native.WS_DECODE_FP8, q, k_cache, v_cache,
                                 k_scale, v_scale, block_tables, seq_lens, float(scale))
    if out is not None:
        return out
    block_tables, seq_lens = _check_pool(k_cache, v_cache, k_scale, v_scale, block_tables,
                                         seq_lens)
    _check_queries(q, k_cache)
    num_seqs, num_q_heads, head_dim = q.shape
    assert seq_lens.shape[0] == num_seqs
    num_blocks, block_size, num_kv_heads, _ = k_cache.shape
    q = _q_ready(q)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if num_seqs == 0 or num_q_heads == 0:
        return out
    lib = _native.load()
    dev = q.device
    st = _native.strides_of
    sizes = (num_seqs, num_q_heads, num_kv_heads, head_dim, block_size, block_tables.shape[1])
    stream = _native.stream_handle(dev)
    with _on_device(dev):
        key = ("decode", dev.index, *sizes)
        nbytes = _ws_sizes.get(key)
        if nbytes is None:
            nbytes = _ws_sizes[key] = lib.pa_decode_fp8_workspace_bytes(*sizes)
        ws, _own = _native.counted_workspace(nbytes, _COUNTER_BYTES, dev, stream,
                                             _native.WS_DECODE_FP8)
        status = lib.pa_decode_fp8(
            q.data_ptr(), st(q), k_cache.data_ptr(), st(k_cache), v_cache.data_ptr(), st(v_cache),
            k_scale.data_ptr(), st(k_scale), v_scale.data_ptr(), st(v_scale),
            block_tables.data_ptr(), st(block_tables), seq_lens.data_ptr(),
            out.data_ptr(), st(out), num_seqs, num_q_heads, num_kv_heads, head_dim, block_size,
            num_blocks, block_tables.shape[1], float(scale), ws, nbytes, stream)
    _native.check(status, "pa_decode_fp8")
    return out


def paged_attention_prefill_fp8(
    q: torch.Tensor,                # [num_tokens, num_q_heads, head_dim] fp16
    k_cache: torch.Tensor,          # [num_blocks, block_size, num_kv_heads, head_dim] float8_e4m3fn
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,          # [num_blocks, num_kv_heads] fp32
    v_scale: torch.Tensor,
    block_tables: torch.Tensor,     # [num_seqs, max_blocks_per_seq] int32
    seq_lens: torch.Tensor,         # [num_seqs] int32: context length after the new tokens
    query_start_loc: torch.Tensor,  # [num_seqs + 1] int32: first q row of each sequence
    max_query_len: int,
    scale: float,
) -> torch.Tensor:
    """Causal attention of each sequence's new tokens over the 8-bit pool.

    paged_attention_prefill on K and V rows = code * scale[block, head]: for prompts,
    chunks of prompts, and the pass over a few drafted tokens per sequence. The new
    tokens' rows must be in the pool (paged_kv_write_fp8); scale must be positive; rows
    of q that belong to no sequence, or lie past max_query_len, are not written.
    """
    out = _native.direct_counted("prefill_fp8", _native.WS_PREFILL, q, k_cache, v_cache, k_scale,
                                 v_scale, block_tables, seq_lens, query_start_loc,
                                 int(max_query_len), float(scale))
    if out is not None:
        return out
    block_tables, seq_lens = _check_pool(k_cache, v_cache, k_scale, v_scale, block_tables,
                                         seq_lens)
    _check_queries(q, k_cache)
    num_tokens, num_q_heads, head_dim = q.shape
    num_seqs = seq_lens.shape[0]
    query_start_loc = _check_starts(query_start_loc, k_cache, num_seqs)
    max_query_len = int(max_query_len)
    assert 0 <= max_query_len < 2 ** 31
    num_blocks, block_size, num_kv_heads, _ = k_cache.shape
    q = _q_ready(q)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if num_seqs == 0 or num_tokens == 0 or num_q_heads == 0 or max_query_len == 0:
        return out
    lib = _native.load()
    dev = q.device
    st = _native.strides_of
    max_blocks = block_tables.shape[1]
    sizes = (num_seqs, num_q_heads, num_kv_heads, head_dim, block_size, max_blocks, max_query_len)
    stream = _native.stream_handle(dev)
    with _on_device(dev):
        key = ("prefill", dev.index, *sizes)
        nbytes = _ws_sizes.get(key)
        if nbytes is None:
            nbytes = _ws_sizes[key] = lib.pa_prefill_attention_fp8_workspace_bytes(*sizes)
        ws, _own = _native.counted_workspace(nbytes, _COUNTER_BYTES, dev, stream,
                                             _native.WS_PREFILL)
        status = lib.pa_prefill_attention_fp8(
            q.data_ptr(), st(q), k_cache.data_ptr(), st(k_cache), v_cache.data_ptr(), st(v_cache),
            k_scale.data_ptr(), st(k_scale), v_scale.data_ptr(), st(v_scale),
            block_tables.data_ptr(), st(block_tables), seq_lens.data_ptr(),
            query_start_loc.data_ptr(), max_query_len, out.data_ptr(), st(out),
            num_seqs, num_tokens, num_q_heads, num_kv_heads, head_dim, block_size, num_blocks,
            max_blocks, float(scale), ws, nbytes, stream)
    _native.check(status, "pa_prefill_attention_fp8")
    return out
