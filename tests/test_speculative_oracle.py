"""The verification oracle, and the entry point's refusals before any launch (no GPU)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from engine.kernels import _native
from engine.kernels.speculative import verify_drafts
from oracle.speculative_oracle import pick, verify

S = _native.i64_array


def emitted(draft_given: bool, m: int, run):
    """First emitted token's distribution over a grid of m x m random numbers, and the target's."""
    p = np.array([0.05, 0.4, 0.3, 0.0, 0.25], dtype=np.float32)
    q = np.array([0.3, 0.1, 0.3, 0.2, 0.1], dtype=np.float32)
    u = (np.arange(m, dtype=np.float32) + 0.5) / m
    got = np.zeros(5)
    for x in range(5):
        target = np.broadcast_to(p, (m * m, 2, 5)).copy()
        draft = np.broadcast_to(q, (m * m, 1, 5)).copy() if draft_given else None
        tokens, _ = run(target, draft, np.full((m * m, 1), x), np.repeat(u, m)[:, None], np.tile(u, m))
        freq = np.bincount(tokens[:, 0], minlength=5) / (m * m)
        if not draft_given:
            # A draft chosen with certainty: the target's distribution whatever it was.
            assert np.abs(freq - p).max() <= 2 / m
        got += q[x] * freq
    return got, p


@pytest.mark.parametrize("draft_given", [True, False])
def test_emitted_tokens_follow_the_target(draft_given):
    """Within the grid's 1/m at the acceptance and 1/m at the draw."""
    got, p = emitted(draft_given, 24, verify)
    assert np.abs(got - p).max() <= 2 / 24


def test_pick():
    w = np.array([0.0, 2.0, 0.0, 1.0, 0.0])
    assert [pick(w, u) for u in (0.0, 0.5, 0.6666, 0.6667, 0.9999999, 1.0)] == [1, 1, 1, 3, 3, 3]
    assert pick(np.zeros(4), 0.5) == 0


def _call(lib, seqs=2, k=3, vocab=100, target=16, tstr=S([400, 100, 1]), draft=16, ids=16, u_next=16,
          ws=0, nbytes=0, dstr=S([300, 100, 1])):
    return lib.pa_verify_drafts_f32(target, tstr, draft, dstr, ids, S([3, 1]), 16, S([3, 1]), u_next,
                                    None, 16, 16, seqs, k, vocab, ws, nbytes, None)


def test_argument_errors_before_launch():
    lib = _native.load()
    for bad in (dict(seqs=-1), dict(k=-1), dict(vocab=0), dict(target=0), dict(ids=0), dict(u_next=0),
                dict(tstr=S([400, 100, 2])), dict(dstr=S([400, 100, 2]))):
        assert _call(lib, **bad) == _native.PA_ERR_ARG, bad
        assert lib.pa_last_error()
    assert _call(lib, k=65) == _native.PA_ERR_UNSUPPORTED
    assert _call(lib, seqs=16385) == _native.PA_ERR_UNSUPPORTED
    assert _call(lib) == _native.PA_ERR_WORKSPACE
    assert _call(lib, ws=16, nbytes=lib.pa_verify_drafts_workspace_bytes(2, 100) - 1) == \
        _native.PA_ERR_WORKSPACE
    assert _call(lib, seqs=0, target=0) == _native.PA_OK
    # Counters, then two sums per sequence and 1024 entries of the vocabulary.
    assert lib.pa_verify_drafts_workspace_bytes(5, 151936) == 16384 * 4 + 5 * 149 * 16
    assert lib.pa_verify_drafts_workspace_bytes(16385, 100) == 0


def test_python_call_needs_the_gpu():
    p = torch.ones(1, 2, 5) / 5
    with pytest.raises(AssertionError, match="GPU"):
        verify_drafts(p, p[:, :1], torch.zeros(1, 1, dtype=torch.int64), torch.zeros(1, 1),
                      torch.zeros(1))
