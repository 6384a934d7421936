"""The 64-bit oracle of the 8-bit pool against torch's conversions and its own bounds (no GPU)."""
from __future__ import annotations

import numpy as np
import torch

from oracle import fp8_cache_oracle as oracle

FP8 = torch.float8_e4m3fn


def test_rounding_is_torch_s_conversion():
    """Every finite fp16 value within 448."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.float16)
    x = x[x.isfinite() & (x.abs() <= 448)]
    want = x.float().to(FP8).float()
    assert np.array_equal(oracle.round_e4m3(x.double().numpy()), want.double().numpy())


def test_scale_is_the_smallest_that_holds_the_maximum():
    for a in [0.0, 2.0 ** -24, 448 * 2.0 ** -15, 448 * 2.0 ** -15 * (1 + 2.0 ** -10), 1.0, 1.75, 1.751,
              447.0, 448.0, 449.0, 57344.0, 57376.0, 61440.0]:
        s = oracle.scale_for(a)
        assert a <= 448 * s and (s == 2.0 ** -15 or a > 448 * s / 2)


def test_every_fp16_value_is_held_within_half_a_step_and_stays_an_fp16_number():
    """Relative error at most 2^-4 of the value, or half of e4m3's smallest step at the scale."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.float16)
    x = x[x.isfinite()].double().numpy()
    for v in x[::7]:
        c = float(oracle.clipped(np.array(v)))
        s = oracle.scale_for(abs(c))
        y = float(oracle.round_e4m3(np.array(c / s))) * s
        assert abs(y - c) <= max(2.0 ** -4 * abs(c), 2.0 ** -10 * s)
        assert abs(y) <= 61440 and float(np.float16(y)) == y


def test_write_then_read_and_a_growing_block():
    """Rows written one at a time: the last scale holds all rows, and earlier rows are within
    half a step of it."""
    rng = np.random.default_rng(3)
    bs, hkv, d, n = 4, 2, 8, 11
    x = rng.standard_normal((n, hkv, d)).astype(np.float16).astype(np.float64)
    x *= 2.0 ** np.arange(n)[:, None, None] / 16
    pool = {k: np.full((5, bs, hkv, d), 7.0) for k in ("k", "v")}
    pool |= {k: np.full((5, hkv), 2.0 ** 8) for k in ("k_scale", "v_scale")}
    tables = np.array([[4, 1, 3]])
    for i in range(n):
        oracle.write(pool, x[i:i + 1], -x[i:i + 1], tables, [i + 1], [0, 1], bs)
    key, value = oracle.read(pool, tables, [n], [0, n], bs, n)
    assert np.array_equal(key, -value)
    for blk in range(3):
        rows = x[blk * bs:(blk + 1) * bs]
        for h in range(hkv):
            s = pool["k_scale"][tables[0, blk], h]
            assert s == oracle.scale_for(np.abs(rows[:, h]).max())
            # A value is rounded once; a code that becomes subnormal once more, by half its step.
            off = np.abs(key[blk * bs:(blk + 1) * bs, h] - rows[:, h])
            assert (off <= 2.0 ** -4 * np.abs(rows[:, h]) + 2.0 ** -10 * s).all()


def test_attention_of_one_key_is_its_value():
    pool = {"k": np.ones((2, 4, 1, 8)), "v": np.arange(64.0).reshape(2, 4, 1, 8),
            "k_scale": np.ones((2, 1)), "v_scale": np.full((2, 1), 0.5)}
    q = np.ones((2, 3, 8))
    out = oracle.attention(pool, q, np.array([[1], [0]]), [1, 0], [0, 1, 2], 4, 1.0)
    assert np.array_equal(out[0], np.broadcast_to(pool["v"][1, 0, 0] * 0.5, (3, 8)))
    assert not out[1].any()
