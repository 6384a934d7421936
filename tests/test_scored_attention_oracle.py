"""The scored attention's oracle by hand and against the plain oracle (no GPU)."""
from __future__ import annotations

import numpy as np
import torch

from oracle.paged_attention_oracle import naive_reference_paged_attention
from oracle.scored_attention_oracle import attend, context


def test_by_hand():
    q = np.array([[[2.0]]])
    k = np.array([[[0.5]], [[1.0]], [[-1.0]]])
    v = np.array([[[1.0]], [[10.0]], [[100.0]]])
    s = np.array([1.0, 2.0, -2.0])
    out, _ = attend(q, k, v, [2], [0], [3], 1.0)
    assert np.allclose(out, (np.exp(s) @ [1, 10, 100]) / np.exp(s).sum())
    s = 1.5 * np.tanh(s / 1.5) - 0.25 * np.array([2, 1, 0])
    out, _ = attend(q, k, v, [2], [0], [3], 1.0, 1.5, np.array([0.25]))
    assert np.allclose(out, (np.exp(s) @ [1, 10, 100]) / np.exp(s).sum())
    assert np.allclose(attend(q, k, v, [2], [1], [2], 1.0)[0], 10.0)
    for first, end, pos in ((2, 2, 2), (3, 9, 2), (0, 0, 2), (0, 3, -1)):
        assert not attend(q, k, v, [pos], [first], [end], 1.0)[0].any()


def test_plain_scores_match_the_plain_oracle():
    rng = np.random.default_rng(0)
    kc, vc = (rng.standard_normal((9, 4, 2, 8)).astype(np.float16) for _ in range(2))
    q = rng.standard_normal((1, 4, 8)).astype(np.float16)
    table, n = np.array([5, 1, 8]), 11
    want = naive_reference_paged_attention(torch.from_numpy(q), torch.from_numpy(kc),
                                           torch.from_numpy(vc), [table.tolist()], [n], 0.3,
                                           compute_dtype=torch.float32)
    got, _ = attend(q, context(kc, table, n, 4), context(vc, table, n, 4), [n - 1], [0], [n], 0.3)
    assert np.abs(got - want.double().numpy()).max() < 1e-3
