"""Forks that are refused for a block that is not allocated leave every count as it was."""
from __future__ import annotations

import pytest


@pytest.mark.parametrize("tokens", [12, 11])
@pytest.mark.parametrize("gone", [0, 1, 2])
def test_a_freed_block_in_the_table(gone, tokens):
    """Shared ones, and a partly filled last one (which a copy could be given)."""
    from engine.kernels.cache_blocks import fork_block_table
    from engine.memory.block_allocator import BlockAllocator, BlockTable

    alloc = BlockAllocator(6)
    table = BlockTable(seq_id=0, block_size=4, physical_block_ids=[alloc.allocate() for _ in range(3)],
                       num_tokens=tokens)
    alloc.free(table.physical_block_ids[gone])
    before = dict(alloc.ref_counts)
    with pytest.raises(ValueError, match="not allocated"):
        fork_block_table(table, alloc, [], 2)
    assert alloc.ref_counts == before
