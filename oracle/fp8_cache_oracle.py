"""The 8-bit paged pool in 64 bits: its write, its read and attention over it.

Test infrastructure only (plain numpy loops over sequences, blocks and rows), written from the
definitions: e4m3 rounded to nearest even, one power-of-two scale per (block, kv head).
A pool is a dict of float64 arrays: k, v [blocks, block size, kv heads, dim] hold the codes'
values (not yet scaled), k_scale, v_scale [blocks, kv heads].
"""
from __future__ import annotations

import numpy as np

EXP_MIN, EXP_MAX, MOST = -15, 8, 61440.0


def round_e4m3(x: np.ndarray) -> np.ndarray:
    """float64 values of magnitude at most 448, to the nearest e4m3 value, ties to even."""
    _, e = np.frexp(x)
    step = np.exp2(np.maximum(e - 1, -6) - 3.0)  # normal from 2^-6 on, three bits after the leading one
    return np.rint(x / step) * step


def scale_for(amax: float) -> float:
    """The smallest power of two of [2^-15, 2^8] with amax <= 448 times it."""
    for e in range(EXP_MIN, EXP_MAX + 1):
        if amax <= 448.0 * 2.0 ** e:
            return 2.0 ** e
    raise AssertionError(amax)


def clipped(x: np.ndarray) -> np.ndarray:
    return np.where(np.isnan(x), x, np.clip(x, -MOST, MOST))


def slots(lens, starts, tables, block_size, num_blocks):
    """Per row: (sequence, block id, row in the block), or None for rows without a slot."""
    out = [None] * starts[-1]
    for b, n in enumerate(lens):
        new = starts[b + 1] - starts[b]
        for i in range(new):
            p = n - new + i
            blk = p // block_size
            if p >= 0 and blk < tables.shape[1] and 0 <= tables[b, blk] < num_blocks:
                out[starts[b] + i] = (b, int(tables[b, blk]), p % block_size)
    return out


def write(pool, key, value, tables, lens, starts, block_size) -> None:
    """Writes float64 rows [tokens, kv heads, dim] into the pool."""
    where = slots(lens, starts, tables, block_size, pool["k"].shape[0])
    for name, x in (("k", clipped(key)), ("v", clipped(value))):
        codes, scale = pool[name], pool[name + "_scale"]
        blocks: dict = {}
        for row, w in enumerate(where):
            if w is not None:
                blocks.setdefault(w[:2], []).append((w[2], row))
        for (_, block), rows in blocks.items():
            first = min(r for r, _ in rows)
            for h in range(codes.shape[2]):
                part = np.abs(x[[row for _, row in rows], h])
                unit = scale_for(float(np.nanmax(np.append(part.ravel(), 0.0))))
                if first > 0:
                    unit = max(unit, scale[block, h])
                    if unit > scale[block, h]:
                        codes[block, :first, h] = round_e4m3(
                            codes[block, :first, h] * (scale[block, h] / unit))
                for r, row in rows:
                    codes[block, r, h] = round_e4m3(x[row, h] / unit)
                scale[block, h] = unit


def read(pool, tables, lens, starts, block_size, num_tokens):
    """(key, value) rows, zeros where there is no slot."""
    hkv, d = pool["k"].shape[2:]
    where = slots(lens, starts, tables, block_size, pool["k"].shape[0])
    out = []
    for name in ("k", "v"):
        y = np.zeros((num_tokens, hkv, d))
        for row, w in enumerate(where):
            if w is not None:
                y[row] = pool[name][w[1], w[2]] * pool[name + "_scale"][w[1]][:, None]
        out.append(y)
    return out


def attention(pool, q, tables, lens, starts, block_size, scale, bound=False):
    """Causal attention of each sequence's rows over its positions 0 .. their own; rows at
    negative positions are zeros. Lengths are cut to the table's width and block ids to the pool.

    With `bound` also how far a kernel may be off that sums in fp32 and rounds probabilities p
    and outputs o to fp16 (half a step of a value x: 2^-11 |x|). Its weights are off by a factor
    1 + e each, and their sum with them, so o is off by at most sum_t w_t |e_t| |v_t - o|, with
    |e| <= 2^-11 (rounded p) + 2 (D + 8) 2^-24 S (a score's fp32 sum of D products and its
    exponential; S the largest scale * sum |q_i| |k_i|) + (L / 32 + 64) 2^-24 (sums over tokens
    by chunks of 32, wavefronts and splits); then its own rounding, and fp16's smallest step.
    """
    rows, hq, d = q.shape
    blocks, _, hkv, _ = pool["k"].shape
    out = np.zeros((rows, hq, d))
    tol = np.zeros((rows, hq, d))
    for b, n in enumerate(lens):
        n = max(0, min(n, tables.shape[1] * block_size))
        ids = np.clip(tables[b, :-(-n // block_size)], 0, blocks - 1)
        k, v = ((pool[c][ids] * pool[c + "_scale"][ids][:, None, :, None]
                 ).reshape(-1, hkv, d)[:n] for c in ("k", "v"))
        new = starts[b + 1] - starts[b]
        for i in range(new):
            pos = n - new + i
            if pos < 0:
                continue
            for h in range(hq):
                g = h // (hq // hkv)
                s = (k[:pos + 1, g] @ q[starts[b] + i, h]) * scale
                p = np.exp(s - s.max())
                w = p / p.sum()
                o = out[starts[b] + i, h] = w @ v[:pos + 1, g]
                if bound:
                    big = (np.abs(k[:pos + 1, g]) @ np.abs(q[starts[b] + i, h])).max() * abs(scale)
                    e = 2.0 ** -11 + (2 * (d + 8) * big + pos / 32 + 64) * 2.0 ** -24
                    around = w @ np.abs(v[:pos + 1, g] - o)
                    tol[starts[b] + i, h] = e * around + 2.0 ** -11 * np.abs(o) + 2.0 ** -24
    return (out, tol) if bound else out
