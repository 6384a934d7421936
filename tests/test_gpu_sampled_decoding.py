"""Sampling, forks, scored attention and verification together, as they are used (needs an MI355X).

Tokens have to equal the 64-bit oracle's on the same logits (or probabilities); attention stays
within the bounds of its own tests; a captured run repeats the eager one's bits.
"""
from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from engine.kernels.cache_blocks import fork_block_table, paged_copy_blocks
from engine.kernels.paged_attention_integration import KernelPagedManualDecode, paged_kv_write
from engine.kernels.sampling import sample_tokens, sampling_probs
from engine.kernels.scored_attention import (paged_attention_decode_scored,
                                             paged_attention_prefill_scored)
from engine.kernels.speculative import verify_drafts
from engine.memory.block_allocator import BlockAllocator, BlockTable
from oracle.sampling_oracle import sample
from oracle.speculative_oracle import verify
from _scored import Pool, check_decode, check_prefill, slopes_of
from test_gpu_decode_step import LOGIT_TOL, TINY, make_model

pytestmark = pytest.mark.gpu


def start(runner, prompt):
    bt = BlockTable(seq_id=0, block_size=runner.block_size)
    bt.physical_block_ids = [runner.allocator.allocate()
                             for _ in range(-(-len(prompt) // runner.block_size))]
    bt.num_tokens = len(prompt)
    seq = SimpleNamespace(seq_id=0, prompt_token_ids=list(prompt), block_table=bt, num_cached_tokens=0,
                          last_token_id=None, generated_ids=[], last_logits=None, last_logit_margin=None)
    seq.last_token_id = runner.prefill(seq)
    return seq


def grow(runner, seqs):
    for s in seqs:
        if s.block_table.num_tokens // runner.block_size >= len(s.block_table.physical_block_ids):
            s.block_table.physical_block_ids.append(runner.allocator.allocate())


@pytest.mark.parametrize("graphs", [False, True])
@torch.inference_mode()
def test_samples_of_a_prompt(cuda_device, graphs):
    """Three samples of one prompt: forked, each with its own settings and numbers, in batched
    steps across a block border; each step's tokens from that step's logits."""
    model = make_model(TINY, 5, cuda_device)
    runner = KernelPagedManualDecode(model, num_blocks=64, device=str(cuda_device), use_graphs=graphs)
    rng = np.random.default_rng(6)
    first = start(runner, rng.integers(0, 512, 41).tolist())
    tables = fork_block_table(first.block_table, runner.allocator,
                              [*runner.pool.k_cache, *runner.pool.v_cache], 2)
    assert [t.physical_block_ids[:2] for t in tables] == [first.block_table.physical_block_ids[:2]] * 2
    seqs = [first] + [SimpleNamespace(seq_id=1 + i, block_table=t, last_token_id=first.last_token_id,
                                      last_logits=None, last_logit_margin=None)
                      for i, t in enumerate(tables)]
    settings = dict(temperature=[0.7, 1.3, 0.0], top_k=[0, 40, 0], top_p=[0.9, 1.0, 1.0])
    on_gpu = {k: torch.tensor(v, dtype=torch.int32 if k == "top_k" else torch.float32, device=cuda_device)
              for k, v in settings.items()}
    for step in range(12):
        grow(runner, seqs)
        u = torch.from_numpy(rng.random(3, dtype=np.float32)).to(cuda_device)
        tokens = runner.decode_step(seqs, sampler=lambda z: sample_tokens(z, u, **on_gpu))
        if step == 0:  # the same context, in blocks of their own
            for s in seqs[1:]:
                assert (s.last_logits.float() - first.last_logits.float()).abs().max() <= LOGIT_TOL
        for i, s in enumerate(seqs):
            own = {k: float(np.float32(v[i])) if k != "top_k" else v[i] for k, v in settings.items()}
            want, gap = sample(s.last_logits.double().cpu().numpy(), float(u[i]), **own)
            assert tokens[i] == want or 0 < gap <= 512 * 2.0 ** -44, (step, i)
            s.last_token_id = tokens[i]
    # Without a sampler the step is the greedy one.
    grow(runner, seqs)
    tokens = runner.decode_step(seqs)
    assert tokens == [int(s.last_logits.argmax()) for s in seqs]
    with pytest.raises(AssertionError, match="must return 3 tokens"):
        grow(runner, seqs)
        runner.decode_step(seqs, sampler=lambda z: z.argmax(-1)[:1])


def test_forks_and_drafts_with_scores(cuda_device):
    """A context forked with its last block copied; drafts written and attended by a capped, biased
    and windowed model, verified from sampled distributions, and the next token's decode."""
    hq, hkv, d, bs, n, k, vocab = 8, 2, 64, 16, 37, 3, 1500
    pool = Pool([n + k + 1] * 3, hkv, d, bs, cuda_device, seed=3, width=8)
    alloc = BlockAllocator(pool.blocks)
    table = BlockTable(seq_id=0, block_size=bs)
    table.physical_block_ids = [alloc.allocate() for _ in range(3)]
    table.num_tokens = n
    before = [t[table.physical_block_ids].clone() for t in (pool.k, pool.v)]
    tables = [table] + fork_block_table(table, alloc, [pool.k, pool.v], 2)
    for i, t in enumerate(tables):
        pool.table[i] = 0
        pool.table[i, :3] = t.physical_block_ids
    pool.tables = torch.from_numpy(pool.table).to(cuda_device)
    rows = n % bs
    for t in tables[1:]:
        for x, old in zip((pool.k, pool.v), before):
            assert torch.equal(x[t.physical_block_ids], old)
    g = torch.Generator(device=cuda_device).manual_seed(4)

    def new(*shape, dtype=torch.float16):
        return torch.randn(shape, generator=g, device=cuda_device).to(dtype)

    kk, vv = new(3 * (k + 1), hkv, d), new(3 * (k + 1), hkv, d)
    for i in range(k + 1):  # each sequence's drafts, a token at a time
        paged_kv_write(kk[i::k + 1], vv[i::k + 1], pool.k, pool.v, pool.tables,
                       torch.full((3,), n + i + 1, dtype=torch.int32, device=cuda_device))
    for x, old in zip((pool.k, pool.v), before):  # the original's own context is as it was
        assert torch.equal(x[table.physical_block_ids[:2]], old[:2])
        assert torch.equal(x[table.physical_block_ids[2]][:rows], old[2][:rows])
    q = pool.queries(3 * (k + 1), hq)
    slopes = slopes_of(hq, cuda_device)
    out = check_prefill(pool, q, [k + 1] * 3, d ** -0.5, softcap=20.0, slopes=slopes, window=24)
    head = 0.3 * new(hq * d, vocab, dtype=torch.float32)
    logits = (out.float().view(3, k + 1, hq * d) @ head).contiguous()
    settings = dict(temperature=0.8, top_k=30, top_p=0.95)
    p = sampling_probs(logits, **settings)
    noisy = (logits[:, :k] + new(3, k, vocab, dtype=torch.float32)).contiguous()
    draft = sampling_probs(noisy, **settings)
    u = torch.rand(3, k, generator=g, device=cuda_device)
    ids = sample_tokens(noisy, u, **settings)
    assert (draft.gather(2, ids[..., None]) > 0).all()
    accept, last = (torch.rand(s, generator=g, device=cuda_device) for s in ((3, k), (3,)))
    tokens, accepted = verify_drafts(p, draft, ids, accept, last)
    want = verify(*(x.cpu().numpy() for x in (p, draft, ids, accept, last)))
    assert np.array_equal(tokens.cpu().numpy(), want[0])
    assert np.array_equal(accepted.cpu().numpy(), want[1])
    # The drafts that were refused are taken back; the contexts differ in length now.
    pool.lens = [n + 1 + int(a) for a in accepted.cpu()]
    pool.seq_lens = pool.ints(pool.lens)
    check_decode(pool, pool.queries(3, hq, seed=9), d ** -0.5, softcap=20.0, slopes=slopes, window=24)


@torch.inference_mode()
def test_captured_run(cuda_device):
    """The whole chain in one graph, replayed over other inputs, with eager calls in between."""
    hq, hkv, d, bs, k, vocab = 8, 2, 64, 16, 2, 33000
    pool = Pool([2300, 17, 640], hkv, d, bs, cuda_device, seed=8)
    slopes = slopes_of(hq, cuda_device)
    head = 0.3 * torch.randn(hq * d, vocab, device=cuda_device, dtype=torch.float32)
    src = pool.ints([int(pool.table[0, 0]), int(pool.table[2, 3])])
    spare = sorted(set(range(pool.blocks)) - {int(x) for r, n in zip(pool.table, pool.lens)
                                             for x in r[:-(-n // bs)]})
    dst = pool.ints(spare[:2])
    loc = pool.ints([0, k + 1, 2 * k + 2, 3 * k + 3])
    q1, q2 = pool.queries(3, hq), pool.queries(3 * (k + 1), hq)
    u, accept = torch.rand(3, device=cuda_device), torch.rand(3, k, device=cuda_device)
    pooled = (pool.k, pool.v, pool.tables, pool.seq_lens)

    def run():
        paged_copy_blocks([pool.k, pool.v], src, dst)
        a = paged_attention_decode_scored(q1, *pooled, d ** -0.5, softcap=30.0, alibi_slopes=slopes)
        b = paged_attention_prefill_scored(q2, *pooled, loc, k + 1, d ** -0.5, softcap=30.0, window=100)
        z = (a.float().view(3, -1) @ head).contiguous()
        tokens = sample_tokens(z, u, temperature=1.1, top_p=0.97)
        p = sampling_probs((b.float().view(3, k + 1, -1) @ head).contiguous(), top_k=50)
        ids = tokens[:, None].expand(3, k).contiguous()
        return (a, b, tokens, p, *verify_drafts(p, None, ids, accept, u), pool.k[dst.long()])

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        held = run()
    for turn in range(4):
        g = torch.Generator(device=cuda_device).manual_seed(turn)
        for x in (q1, q2):
            x.copy_(2 * torch.randn(x.shape, generator=g, device=cuda_device))
        for x in (u, accept):
            x.copy_(torch.rand(x.shape, generator=g, device=cuda_device))
        graph.replay()
        got = [x.clone() for x in held]
        torch.cuda.synchronize()
        for x, want in zip(got, run()):
            assert torch.equal(x, want), turn
