"""decode_step's sampler on the host: errors leave the sequences as they were, and what it does
to its argument stays there."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

VOCAB = 8


class Model(torch.nn.Module):
    """Logits of 0 .. 7 in a row's order, turned by its token; no attention."""

    config = SimpleNamespace(num_hidden_layers=1, num_key_value_heads=2, head_dim=64, hidden_size=128,
                             num_attention_heads=2)

    def __init__(self):
        super().__init__()
        self.embedding = torch.nn.Embedding(VOCAB, 4)
        self.steps = 0

    def get_input_embeddings(self):
        return self.embedding

    def forward(self, input_ids, position_ids, use_cache):
        self.steps += 1
        rows = [torch.arange(VOCAB, dtype=torch.float32).roll(int(t)) for t in input_ids[:, 0]]
        return SimpleNamespace(logits=torch.stack(rows)[:, None, :])


@pytest.fixture
def batch():
    from engine.kernels.paged_attention_integration import KernelPagedManualDecode
    from engine.memory.block_allocator import BlockTable

    runner = KernelPagedManualDecode(Model(), block_size=16, num_blocks=4, device="cpu", use_graphs=False)
    return runner, [SimpleNamespace(seq_id=i, block_table=BlockTable(i, 16, [runner.allocator.allocate()], 3 + i),
                                    last_token_id=2 * i, last_logits=None, last_logit_margin=None)
                    for i in range(3)]


def raising(z):
    raise KeyError("grammar")


@pytest.mark.parametrize("sampler,error,message", [
    (raising, KeyError, "grammar"),
    (lambda z: z.argmax(-1)[:2], AssertionError, "must return 3 tokens"),
    (lambda z: [1, 2, 3], AssertionError, "must return 3 tokens"),
    (lambda z: z.argmax(-1).to("meta"), AssertionError, "on cpu"),
    (lambda z: z[:, 0] * float("nan"), ValueError, "NaN"),
])
def test_errors_leave_the_sequences_as_they_were(batch, sampler, error, message):
    runner, seqs = batch
    with pytest.raises(error, match=message):
        runner.decode_step(seqs, sampler=sampler)
    assert [s.block_table.num_tokens for s in seqs] == [3, 4, 5]
    assert all(s.last_logits is None and s.last_logit_margin is None for s in seqs)
    # The step can be taken again.
    assert runner.decode_step(seqs, sampler=lambda z: z.argmin(-1)) == [0, 2, 4]
    assert [s.block_table.num_tokens for s in seqs] == [4, 5, 6] and runner.model.steps == 2


def test_a_sampler_may_write_its_argument(batch):
    runner, seqs = batch

    def sampler(z):
        z.div_(0.5)
        z[:, 4] = float("inf")
        return z.argmax(-1)

    assert runner.decode_step(seqs, sampler=sampler) == [4, 4, 4]
    for i, s in enumerate(seqs):
        assert torch.equal(s.last_logits, torch.arange(VOCAB, dtype=torch.float32).roll(2 * i))
        assert s.last_logit_margin == 1.0
