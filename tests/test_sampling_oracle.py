"""The sampling oracle against small cases worked by hand, and a second formulation (no GPU)."""
from __future__ import annotations

import numpy as np
import pytest

from oracle.sampling_oracle import kept_weights, probabilities, sample

Z = np.log(np.array([0.1, 0.4, 0.2, 0.3]))


def kept(**settings):
    return np.flatnonzero(kept_weights(Z, **settings)).tolist()


def test_by_hand():
    assert np.allclose(probabilities(Z), [0.1, 0.4, 0.2, 0.3])
    assert kept(top_k=2) == [1, 3]
    assert kept(top_p=0.69) == [1, 3] and kept(top_p=0.71) == [1, 2, 3]
    assert kept(top_p=0.0) == [1] and kept(top_k=1) == [1]
    assert kept(min_p=0.6) == [1, 3] and kept(min_p=2.0) == [1]
    assert kept(top_k=3, top_p=0.7) == [1, 3]  # 0.7 of 0.9
    assert kept(temperature=0.0) == [1]
    assert np.allclose(probabilities(Z, temperature=0.5), np.array([1, 16, 4, 9]) / 30)
    for u, token in ((0.0, 0), (0.05, 0), (0.15, 1), (0.6, 2), (0.75, 3), (1.0, 3), (np.nan, 3)):
        assert sample(Z, u)[0] == token
    assert sample(Z, 0.5, top_k=2)[0] == 1 and sample(Z, 0.6, top_k=2)[0] == 3


def test_ties_and_odd_values():
    z = np.array([1.0, 2.0, 2.0, np.nan, 2.0, -np.inf])
    assert np.flatnonzero(kept_weights(z, top_k=2)).tolist() == [1, 2]
    assert np.flatnonzero(kept_weights(z)).tolist() == [0, 1, 2, 4]
    assert np.flatnonzero(kept_weights(np.array([0.0, np.inf, 5.0, np.inf]))).tolist() == [1, 3]
    dead = np.array([-np.inf, np.nan])
    assert not kept_weights(dead).any() and sample(dead, 0.5)[0] == 0
    assert np.flatnonzero(kept_weights(np.array([-0.0, 0.0, -1.0]), top_k=1)).tolist() == [0]


@pytest.mark.parametrize("settings", [{}, {"top_k": 7}, {"top_p": 0.8}, {"min_p": 0.1},
                                      {"top_k": 30, "top_p": 0.7, "min_p": 0.02, "temperature": 1.7}])
def test_frequencies(settings):
    z = 2 * np.random.default_rng(0).standard_normal(50)
    p = probabilities(z, **settings)
    grid = (np.arange(20000) + 0.5) / 20000
    tokens = [sample(z, u, **settings)[0] for u in grid]
    assert np.abs(np.bincount(tokens, minlength=50) / 20000 - p).max() < 1e-4
