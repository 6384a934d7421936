"""Sampling from a decode step's logits: temperature, top-k, top-p and min-p.

No counterpart in the reference, whose decode step selects greedily
(engine/kernels/paged_attention_integration.py:636-651). Random numbers are the caller's:
the same logits, settings and numbers give the same tokens. sampling_probs gives the
distributions that verify_drafts takes for drafted tokens under the same settings.
"""
from __future__ import annotations

from typing import Tuple, Union

import torch

from . import _native
from .paged_attention import _on_device

__all__ = [
    "sample_tokens",
    "sampling_probs",
]

_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
# Bytes of the arrival counters at the head of the workspace (16384 ints).
_COUNTER_BYTES = 65536

Setting = Union[float, torch.Tensor]


def _setting(name: str, x: Setting, dtype: torch.dtype, logits: torch.Tensor) -> Tuple:
    """(tensor or None, number for all) of a setting."""
    if not isinstance(x, torch.Tensor):
        if dtype == torch.int32:
            assert int(x) == x, f"{name} must be a whole number, got {x}"
            # (Numbers beyond 32 bits mean what the ends do: off, or all.)
            return None, max(-2 ** 31 + 1, min(2 ** 31 - 1, int(x)))
        return None, float(x)
    assert x.is_cuda and x.dtype == dtype, f"{name} must be {dtype} on the GPU, got {x.dtype}"
    _native.same_device(x, logits)
    assert x.shape == (logits.shape[0],), (
        f"{name} must have one entry per sequence ({logits.shape[0]}), got {tuple(x.shape)}")
    return x.contiguous(), 0


def _arguments(logits, temperature, top_k, top_p, min_p):
    """(logits with unit vocabulary stride, strides, settings)."""
    assert logits.is_cuda, "sampling runs on the GPU only"
    assert logits.dtype in _TYPES, f"logits must be fp16, bf16 or fp32, got {logits.dtype}"
    assert logits.dim() in (2, 3) and logits.shape[-1] > 0, (
        f"logits must be [num_seqs, vocab] or [num_seqs, rows, vocab], got {tuple(logits.shape)}")
    settings = [_setting("temperature", temperature, torch.float32, logits),
                _setting("top_k", top_k, torch.int32, logits),
                _setting("top_p", top_p, torch.float32, logits),
                _setting("min_p", min_p, torch.float32, logits)]
    if logits.stride(-1) != 1:
        logits = logits.contiguous()
    x = logits if logits.dim() == 3 else logits.unsqueeze(1)
    return x, settings


def _call(name, x, dev, settings, before, out):
    """Launches pa_<name> on [seqs, rows, vocab] logits x."""
    lib = _native.load()
    seqs, rows, vocab = x.shape
    stream = _native.stream_handle(dev)
    numbers = [v for t, n in settings for v in (None if t is None else t.data_ptr(), n)]
    with _on_device(dev):
        nbytes = lib.pa_sample_workspace_bytes(seqs, rows, vocab)
        ws, _own = _native.counted_workspace(nbytes, _COUNTER_BYTES, dev, stream, _native.WS_SAMPLE)
        status = getattr(lib, name)(
            x.data_ptr(), _TYPES[x.dtype], _native.strides_of(x), *before, *numbers, out.data_ptr(),
            seqs, rows, vocab, ws, nbytes, stream)
    _native.check(status, name)


def sample_tokens(
    logits: torch.Tensor,        # [num_seqs, vocab] or [num_seqs, rows, vocab], fp16, bf16 or fp32
    u: torch.Tensor,             # logits.shape[:-1], fp32 random numbers of [0, 1)
    temperature: Setting = 1.0,  # each a number for all, or [num_seqs] (fp32, top_k int32)
    top_k: Setting = 0,
    top_p: Setting = 1.0,
    min_p: Setting = 0.0,
) -> torch.Tensor:
    """One token id per row of logits, int64 [logits.shape[:-1]].

    With weights w = exp((z - max z) / temperature) and the entries ordered by logit, largest
    first, equal ones by index: the first top_k stay (0: all), of them the shortest beginning
    that weighs at least top_p of their sum (one entry at least; 1: all), of those the ones
    with w >= min_p. The token is the first index, in the vocabulary's order, whose cumulative
    kept weight exceeds u times their sum. A temperature of 0 takes the first of the largest
    logits. NaN logits count as -inf, which has no weight; a row without any weight gives 0;
    u of 1 and more, or NaN, the last index with a weight.

    Weights and sums are in 64 bits (units of 2^-44 of the largest weight). At most 16384 rows
    of 2^19 logits. One launch, and two more where a row can have a long list (more than 2048
    logits); asynchronous on the current stream; no host synchronisation; capturable into a HIP
    graph.
    """
    out = _native.direct_counted("sample", _native.WS_SAMPLE, logits, u, temperature, top_k, top_p,
                                 min_p)
    if out is not None:
        return out
    x, settings = _arguments(logits, temperature, top_k, top_p, min_p)
    assert u.is_cuda and u.dtype == torch.float32
    _native.same_device(logits, u)
    assert u.shape == logits.shape[:-1], (
        f"u must be {tuple(logits.shape[:-1])}, got {tuple(u.shape)}")
    tokens = torch.empty(u.shape, dtype=torch.int64, device=u.device)
    if tokens.numel() == 0:
        return tokens
    u2 = u if u.dim() == 2 else u.unsqueeze(1)
    _call("pa_sample_tokens", x, u.device, settings, (u2.data_ptr(), _native.strides_of(u2)), tokens)
    return tokens


def sampling_probs(
    logits: torch.Tensor,        # [num_seqs, vocab] or [num_seqs, rows, vocab], fp16, bf16 or fp32
    temperature: Setting = 1.0,  # each a number for all, or [num_seqs] (fp32, top_k int32)
    top_k: Setting = 0,
    top_p: Setting = 1.0,
    min_p: Setting = 0.0,
) -> torch.Tensor:
    """The distributions that sample_tokens draws from, fp32 of logits' shape.

    w / sum for the entries that its settings keep, 0 for all others (and for a row without
    any weight). The target_probs and draft_probs of verify_drafts. One launch more
    than sample_tokens, and otherwise as it.
    """
    out = _native.direct_counted("probabilities", _native.WS_SAMPLE, logits, temperature, top_k,
                                 top_p, min_p)
    if out is not None:
        return out
    x, settings = _arguments(logits, temperature, top_k, top_p, min_p)
    probs = torch.empty(logits.shape, dtype=torch.float32, device=logits.device)
    if probs.numel() == 0:
        return probs
    _call("pa_sampling_probs", x, logits.device, settings, (), probs)
    return probs
