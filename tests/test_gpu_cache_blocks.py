"""Copies of pool blocks, bit for bit against indexing on the CPU (needs an MI355X)."""
from __future__ import annotations

import pytest
import torch

from engine.kernels.cache_blocks import fork_block_table, paged_copy_blocks
from engine.memory.block_allocator import BlockAllocator, BlockTable

pytestmark = pytest.mark.gpu


def pool(shape, count, device, dtype=torch.float16, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    out = []
    for _ in range(count):
        bits = torch.randint(0, 256, (*shape[:-1], shape[-1] * dtype.itemsize), generator=g,
                             device=device, dtype=torch.uint8)
        out.append(bits.view(dtype))
    return out


def bits(t):
    return t.contiguous().view(torch.uint8).cpu()


def ids(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def check(caches, src, dst):
    want = []
    for t in caches:
        x = t.cpu().contiguous().view(torch.uint8).reshape(t.shape[0], -1).clone()
        for a, b in zip(src.tolist(), dst.tolist()):
            if 0 <= a < t.shape[0] and 0 <= b < t.shape[0]:
                x[b] = x[a]
        want.append(x)
    paged_copy_blocks(caches, src, dst)
    for t, x in zip(caches, want):
        assert torch.equal(bits(t).reshape(t.shape[0], -1), x)


@pytest.mark.parametrize("shape", [(40, 16, 2, 64), (40, 16, 8, 128), (33, 8, 1, 32), (40, 32, 16, 64),
                                   (20, 16, 3, 40), (24, 2), (24, 1), (24, 3), (24, 7, 5)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float8_e4m3fn, torch.float32])
def test_matches_indexing(cuda_device, shape, dtype):
    perm = torch.randperm(shape[0], generator=torch.Generator().manual_seed(1)).tolist()
    half = shape[0] // 2
    for n in (1, 3, half):
        check(pool(shape, 3, cuda_device, dtype), ids(perm[:n], cuda_device),
              ids(perm[half:half + n], cuda_device))


def test_one_source_of_many_and_ids_out_of_range(cuda_device):
    caches = pool((30, 16, 2, 64), 4, cuda_device)
    check(caches, ids([3] * 9, cuda_device), ids(list(range(10, 19)), cuda_device))
    check(caches, ids([-1, 30, 5, 6, 2 ** 31 - 1, -2 ** 31, 8], cuda_device),
          ids([20, 21, 30, -5, 22, 23, 24], cuda_device))
    check(caches, ids([7, 9], cuda_device), ids([7, 10], cuda_device))  # onto itself


def test_pools_of_many_layers_and_mixed_tensors(cuda_device):
    """More tensors than one launch takes; codes and scales of an 8-bit pool; views."""
    caches = pool((12, 16, 2, 64), 200, cuda_device, torch.float8_e4m3fn)
    caches += pool((12, 2), 100, cuda_device, torch.float32)
    merged = pool((12, 2, 16, 2, 64), 1, cuda_device)[0]
    caches += [merged[:, 0], merged[:, 1]]
    odd = pool((12, 4099), 1, cuda_device, torch.uint8)[0]
    caches += [odd[:, 1:4098], odd[:, 4098:]]
    check(caches, ids([0, 1, 2, 1], cuda_device), ids([8, 11, 9, 10], cuda_device))


def test_strided_ids_and_large_pools(cuda_device):
    pairs = ids([[0, 5], [1, 6], [2, 7]], cuda_device)
    check(pool((9, 16, 2, 64), 2, cuda_device), pairs[:, 0], pairs[:, 1])
    big = torch.zeros(70000, 16, 16, 128, dtype=torch.float16, device=cuda_device)  # past 2^31 elements
    big[0] = 3
    big[69998] = 5
    paged_copy_blocks([big], ids([0, 69998], cuda_device), ids([69999, 40000], cuda_device))
    assert (big[69999] == 3).all() and (big[40000] == 5).all() and (big[69997] == 0).all()


def test_captured(cuda_device):
    with torch.inference_mode():
        caches = pool((20, 16, 2, 64), 6, cuda_device)
        src, dst = ids([1, 2], cuda_device), ids([10, 11], cuda_device)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            paged_copy_blocks(caches, src, dst)
        for i in range(3):
            src.copy_(ids([i, i + 3], cuda_device))
            dst.copy_(ids([12 + i, 16 + i], cuda_device))
            before = [t.clone() for t in caches]
            graph.replay()
            paged_copy_blocks(before, src, dst)
            for t, x in zip(caches, before):
                assert torch.equal(bits(t), bits(x))


def test_nothing_and_refusals(cuda_device):
    caches = pool((10, 16, 2, 64), 2, cuda_device)
    one = ids([1], cuda_device)
    paged_copy_blocks([], one, one)
    paged_copy_blocks(caches, one[:0], one[:0])
    for bad in (lambda: paged_copy_blocks(caches, one.long(), one),
                lambda: paged_copy_blocks(caches, one, ids([1, 2], cuda_device)),
                lambda: paged_copy_blocks(caches, one.cpu(), one),
                lambda: paged_copy_blocks([caches[0], caches[1][:5]], one, one),
                lambda: paged_copy_blocks([caches[0].transpose(1, 2)], one, one),
                lambda: paged_copy_blocks([caches[0][:1].expand(5, -1, -1, -1)], one, one),
                lambda: paged_copy_blocks([caches[0].cpu()], one, one)):
        with pytest.raises(AssertionError):
            bad()


def test_fork_of_a_table(cuda_device):
    caches = pool((20, 16, 2, 64), 4, cuda_device)
    alloc = BlockAllocator(20)
    table = BlockTable(seq_id=4, block_size=16)
    table.physical_block_ids = [alloc.allocate() for _ in range(4)]
    table.num_tokens = 37  # two full blocks, five tokens of a third, one block ahead
    copies = fork_block_table(table, alloc, caches, 3)
    assert [t.num_tokens for t in copies] == [37] * 3
    for t in copies:
        assert t.physical_block_ids[:2] == table.physical_block_ids[:2] and len(t.physical_block_ids) == 3
        for c in caches:
            assert torch.equal(bits(c[t.physical_block_ids[2]]), bits(c[table.physical_block_ids[2]]))
    last = [t.physical_block_ids[2] for t in copies] + [table.physical_block_ids[2]]
    assert len(set(last)) == 4 and all(alloc.ref_counts[b] == 1 for b in last)
    assert [alloc.ref_counts[b] for b in table.physical_block_ids] == [4, 4, 1, 1]
    for t in copies:
        t.free(alloc)
    assert [alloc.ref_counts[b] for b in table.physical_block_ids] == [1, 1, 1, 1]
    table.num_tokens = 32  # nothing to copy
    free = alloc.num_available()
    assert [t.physical_block_ids for t in fork_block_table(table, alloc, caches, 2)] == [
        table.physical_block_ids[:2]] * 2
    assert alloc.num_available() == free
    table.num_tokens = 40
    counts = dict(alloc.ref_counts)
    with pytest.raises(MemoryError):
        fork_block_table(table, alloc, caches, 100)
    assert alloc.ref_counts == counts
