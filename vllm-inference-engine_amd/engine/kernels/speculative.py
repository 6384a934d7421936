"""Speculative decoding: drafted tokens against the target's probabilities.

No counterpart in the reference, whose decode step selects greedily
(engine/kernels/paged_attention_integration.py:636-651). The target's pass over the
drafts is an ordinary several-token attention over the paged pool
(paged_attention_prefill, or paged_attention_prefill_fp8 for the 8-bit pool);
verify_drafts decides from its probabilities which drafts stay and what follows.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _native
from .paged_attention import _on_device

__all__ = ["verify_drafts"]


def verify_drafts(
    target_probs: torch.Tensor,           # [num_seqs, max_drafts + 1, vocab] fp32
    draft_probs: Optional[torch.Tensor],  # [num_seqs, max_drafts, vocab] fp32, or None
    draft_ids: torch.Tensor,              # [num_seqs, max_drafts] int64
    accept_u: torch.Tensor,               # [num_seqs, max_drafts] fp32 random numbers of [0, 1)
    next_u: torch.Tensor,                 # [num_seqs] fp32 random numbers of [0, 1)
    num_drafts: Optional[torch.Tensor] = None,  # [num_seqs] int32, default max_drafts each
) -> Tuple[torch.Tensor, torch.Tensor]:
    """(tokens [num_seqs, max_drafts + 1] int64, accepted [num_seqs] int32).

    Draft i of a sequence is accepted while accept_u[i] * draft_probs[i, id] <
    target_probs[i, id]; after n accepted ones the next token is drawn by next_u from
    max(target_probs[n] - draft_probs[n], 0), or from target_probs[n] if all drafts were
    accepted (or that difference is 0 everywhere): the first index whose cumulative sum
    exceeds next_u times the whole sum. The emitted tokens then follow the target's
    distribution. draft_probs None: the drafts were chosen with certainty (greedy, or
    looked up), so draft i is accepted with probability target_probs[i, id] and left out
    of the draw if it is not. A row of tokens holds the accepted drafts, the next token,
    then -1.

    The rows need not sum to 1. Sums and products are in 64 bits; a negative weight or
    NaN counts as none; an id outside the vocabulary is not accepted, nor one whose random
    number is NaN; a next_u of 1 and more or NaN takes the last index with a weight. At most 64
    drafts and 16384 sequences. Asynchronous on the current stream; no host
    synchronisation; capturable into a HIP graph.
    """
    out = _native.direct_counted("verify", _native.WS_VERIFY, target_probs, draft_probs, draft_ids,
                                 accept_u, next_u, num_drafts)
    if out is not None:
        return out
    tensors = [target_probs, draft_ids, accept_u, next_u]
    tensors += [t for t in (draft_probs, num_drafts) if t is not None]
    assert all(t.is_cuda for t in tensors), "verify_drafts runs on the GPU only"
    _native.same_device(*tensors)
    assert target_probs.dtype == torch.float32 and target_probs.dim() == 3
    num_seqs, rows, vocab = target_probs.shape
    max_drafts = rows - 1
    assert max_drafts >= 0 and vocab > 0, (
        f"target_probs must be [num_seqs, max_drafts + 1, vocab], got {tuple(target_probs.shape)}")
    if draft_probs is not None:
        assert draft_probs.dtype == torch.float32
        assert draft_probs.shape == (num_seqs, max_drafts, vocab), (
            f"draft_probs must be {(num_seqs, max_drafts, vocab)}, got {tuple(draft_probs.shape)}")
    assert draft_ids.dtype == torch.int64 and draft_ids.shape == (num_seqs, max_drafts)
    assert accept_u.dtype == torch.float32 and accept_u.shape == (num_seqs, max_drafts)
    assert next_u.dtype == torch.float32 and next_u.shape == (num_seqs,)
    if num_drafts is not None:
        assert num_drafts.dtype == torch.int32 and num_drafts.shape == (num_seqs,)
        num_drafts = num_drafts.contiguous()
    if target_probs.stride(2) != 1:
        target_probs = target_probs.contiguous()
    if draft_probs is not None and draft_probs.stride(2) != 1:
        draft_probs = draft_probs.contiguous()
    next_u = next_u.contiguous()

    dev = target_probs.device
    tokens = torch.empty((num_seqs, rows), dtype=torch.int64, device=dev)
    accepted = torch.empty((num_seqs,), dtype=torch.int32, device=dev)
    if num_seqs == 0:
        return tokens, accepted
    lib = _native.load()
    st = _native.strides_of
    stream = _native.stream_handle(dev)
    with _on_device(dev):
        nbytes = lib.pa_verify_drafts_workspace_bytes(num_seqs, vocab)
        ws, _own = _native.counted_workspace(nbytes, 4 * num_seqs, dev, stream, _native.WS_VERIFY)
        status = lib.pa_verify_drafts_f32(
            target_probs.data_ptr(), st(target_probs),
            None if draft_probs is None else draft_probs.data_ptr(),
            None if draft_probs is None else st(draft_probs),
            draft_ids.data_ptr(), st(draft_ids), accept_u.data_ptr(), st(accept_u),
            next_u.data_ptr(), None if num_drafts is None else num_drafts.data_ptr(),
            tokens.data_ptr(), accepted.data_ptr(), num_seqs, max_drafts, vocab, ws, nbytes,
            stream)
    _native.check(status, "pa_verify_drafts_f32")
    return tokens, accepted
