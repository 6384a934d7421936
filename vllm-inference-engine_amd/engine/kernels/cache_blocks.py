"""Blocks of a paged pool copied to other blocks: forks, beams, contexts moved together.

No counterpart in the reference, which shares full blocks by reference counts
(engine/memory/block_allocator.py:143-270) and refuses to write a shared one
(engine/kernels/paged_attention_integration.py:587-592): a fork of a sequence whose last
block is partly filled needs that block copied before either side goes on.
"""
from __future__ import annotations

from typing import Any, List, Sequence

import torch

from . import _native
from .paged_attention import _on_device

__all__ = [
    "paged_copy_blocks",
    "fork_block_table",
]


def paged_copy_blocks(
    caches: Sequence[torch.Tensor],  # each [num_blocks, ...], any type: K, V, scales of the layers
    src_blocks: torch.Tensor,        # [n] int32
    dst_blocks: torch.Tensor,        # [n] int32
) -> None:
    """t[dst_blocks[i]] = t[src_blocks[i]] for every tensor of `caches` and every i.

    Every block is copied bit for bit. The tensors share num_blocks and the device; a
    block's own elements must be contiguous, the distance from block to block may be any.
    Pairs with an id outside [0, num_blocks) are skipped. A block may be the source of
    several pairs; one that is a destination must not be in any other pair (what the blocks
    of such pairs hold afterwards is not defined). One launch for up to 96 tensors, on the
    current stream; no host synchronisation; capturable into a HIP graph, which keeps the
    tensors' addresses.
    """
    caches = list(caches)
    if caches and _native.direct_call("copy_blocks", src_blocks, dst_blocks, caches):
        return
    assert all(t.is_cuda for t in caches) and src_blocks.is_cuda and dst_blocks.is_cuda, (
        "paged_copy_blocks runs on the GPU only")
    _native.same_device(src_blocks, dst_blocks, *caches)
    assert src_blocks.dtype == torch.int32 and dst_blocks.dtype == torch.int32
    assert src_blocks.dim() == 1 and dst_blocks.shape == src_blocks.shape, (
        f"src_blocks {tuple(src_blocks.shape)} and dst_blocks {tuple(dst_blocks.shape)} must be "
        "one list of pairs")
    for t in caches:
        assert t.dim() >= 1 and t.shape[0] == caches[0].shape[0], (
            f"every tensor must have {caches[0].shape[0]} blocks, got {tuple(t.shape)}")
        assert t.shape[0] == 0 or t[0].is_contiguous(), (
            f"a block's elements must be contiguous, got strides {t.stride()}")
        assert t.shape[0] <= 1 or t.stride(0) >= t[0].numel(), "blocks must not overlap"
    pairs = src_blocks.shape[0]
    if not caches or pairs == 0 or caches[0].shape[0] == 0:
        return
    lib = _native.load()
    dev = src_blocks.device
    n = len(caches)
    sizes = [t[0].numel() * t.element_size() for t in caches]
    strides = [max(t.stride(0) * t.element_size(), size) for t, size in zip(caches, sizes)]
    with _on_device(dev):
        status = lib.pa_copy_blocks(
            _native.pointer_array(t.data_ptr() for t in caches), _native.i64_array(strides),
            _native.i64_array(sizes), n, src_blocks.data_ptr(), src_blocks.stride(0),
            dst_blocks.data_ptr(), dst_blocks.stride(0), pairs, caches[0].shape[0],
            _native.stream_handle(dev))
    _native.check(status, "pa_copy_blocks")


def fork_block_table(table: Any, allocator: Any, caches: Sequence[torch.Tensor],
                     copies: int = 1) -> List[Any]:
    """`copies` tables that go on from table's tokens, each on its own: samples of one prompt,
    beams. caches: the pool's K and V of every layer, [*pool.k_cache, *pool.v_cache] (with the
    scales, for an 8-bit pool).

    Full blocks are shared (allocator.fork); a partly filled last block is copied into a
    block of each copy's own (allocator.allocate) in all tensors of `caches`, so that
    decode steps of the copies and of the original never write a shared block. Blocks that
    the table holds beyond its tokens stay its own alone. Raises what allocate() raises when
    blocks run out, fork() for a block that is not allocated, and paged_copy_blocks for the
    caches, with every count as it was.
    """
    full, rest = divmod(table.num_tokens, table.block_size)
    shared = list(table.physical_block_ids[:full])
    assert len(table.physical_block_ids) >= full + (rest > 0), (
        f"a table of {table.num_tokens} tokens needs {full + (rest > 0)} blocks")
    assert copies >= 0
    own: List[int] = []
    forked: List[int] = []
    try:
        last = list(table.physical_block_ids[full:full + 1]) if rest and copies else []
        for b in last + shared * copies:  # (the last one is held while it is copied)
            allocator.fork(b)
            forked.append(b)
        for _ in range(copies if rest else 0):
            own.append(allocator.allocate())
        if own:
            pairs = torch.tensor([last * copies, own], dtype=torch.int32).to(caches[0].device)
            paged_copy_blocks(caches, pairs[0], pairs[1])
    except BaseException:
        for b in own + forked:
            allocator.free(b)
        raise
    for b in last:
        allocator.free(b)
    return [type(table)(seq_id=table.seq_id, block_size=table.block_size,
                        physical_block_ids=shared + own[i:i + 1], num_tokens=table.num_tokens)
            for i in range(copies)]
