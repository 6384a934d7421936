"""Verification of drafted tokens against the 64-bit oracle (needs an MI355X).

Tokens and counts are whole numbers and have to be equal: both sides compare exact 64-bit
products and pick from 64-bit sums, whose order changes them by less than 2^-40 of the whole.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from engine.kernels import _native
from engine.kernels.speculative import verify_drafts
from oracle.speculative_oracle import verify
from test_speculative_oracle import emitted

pytestmark = pytest.mark.gpu


def case(seqs, k, vocab, seed, device, off=0.7):
    g = torch.Generator(device=device).manual_seed(seed)
    logits = 2.5 * torch.randn(seqs, k + 1, vocab, generator=g, device=device)
    p = torch.softmax(logits, dim=-1)
    q = torch.softmax(logits[:, :k] + off * torch.randn(seqs, k, vocab, generator=g, device=device), -1)
    ids = torch.multinomial(q.reshape(seqs * k, vocab), 1, generator=g).view(seqs, k) if k else \
        torch.zeros(seqs, 0, dtype=torch.int64, device=device)
    u = torch.rand(seqs, k, generator=g, device=device)
    return p, q, ids, u, torch.rand(seqs, generator=g, device=device)


def on_host(*tensors):
    return [None if t is None else t.cpu().numpy() for t in tensors]


def check(*args):
    tokens, accepted = verify_drafts(*args)
    want = verify(*on_host(*args))
    assert np.array_equal(accepted.cpu().numpy(), want[1])
    assert np.array_equal(tokens.cpu().numpy(), want[0])
    return want


@pytest.mark.parametrize("seqs,k,vocab", [(1, 4, 151936), (7, 3, 32000), (64, 1, 4096), (9, 8, 4097),
                                          (5, 64, 100), (33, 5, 255), (4, 2, 1), (3, 0, 5000),
                                          (300, 2, 17), (2, 6, 8191), (2, 2, 600001)])
def test_matches_oracle(cuda_device, seqs, k, vocab):
    args = case(seqs, k, vocab, seqs * 100 + k, cuda_device)
    check(*args)
    p, q, ids, u, nxt = args
    check(p, None, ids, u * 0.2, nxt)


@pytest.mark.parametrize("given", [True, False])
def test_counts_of_each_sequence(cuda_device, given):
    """Fewer drafts than columns, none, and counts out of range."""
    p, q, ids, u, nxt = case(40, 6, 1000, 1, cuda_device, off=0.3)
    counts = torch.tensor([(i % 9) - 1 for i in range(40)], dtype=torch.int32, device=cuda_device)
    want = check(p, q if given else None, ids, u * 0.5, nxt, counts)
    assert want[1].max() > (1 if given else 0)


def test_all_accepted_and_none(cuda_device):
    p, q, ids, u, nxt = case(8, 5, 5000, 2, cuda_device)
    assert (check(p, q, ids, torch.zeros_like(u), nxt)[1] == 5).all()
    assert (check(p * 0.001, q, ids, torch.full_like(u, 0.999), nxt)[1] == 0).all()
    # p == q: every u < 1 accepts.
    assert (check(p, p[:, :5].contiguous(), ids, torch.full_like(u, 1 - 2.0 ** -24), nxt)[1] == 5).all()


def test_border_numbers(cuda_device):
    """next_u of 0, the largest below 1, 1 and NaN; equal dyadic weights, where u hits a border."""
    p, q, ids, u, _ = case(6, 2, 9000, 3, cuda_device)
    for x in (0.0, 1 - 2.0 ** -24, 1.0):
        check(p, q, ids, u, torch.full((6,), x, device=cuda_device))
    p = torch.full((64, 1, 16384), 2.0 ** -14, device=cuda_device)
    nxt = torch.arange(64, device=cuda_device).float() / 64
    want = check(p, None, torch.zeros(64, 0, dtype=torch.int64, device=cuda_device),
                 torch.zeros(64, 0, device=cuda_device), nxt)
    assert (want[0][:, 0] == np.arange(64) * 256).all()


def test_rows_without_weight_nan_and_negative_numbers(cuda_device):
    p, q, ids, u, nxt = case(6, 2, 5000, 4, cuda_device)
    u = torch.ones_like(u)
    q[0] = 2.0                     # p <= q everywhere: the target's own row
    p[1] = 0.0                     # nothing anywhere: index 0
    p[2, :, ::2] = float("nan")
    p[3, :, 1::2] = -1.0
    p[4] = 0.0
    p[4, :, 4321] = 1e-30          # one entry
    ids[5, 0] = 5000               # outside the vocabulary: not accepted
    ids[5, 1] = -1
    for draft in (q, None):
        want = check(p, draft, ids, u, nxt)
        assert want[0][1, 0] == 0 and want[0][4, 0] == 4321 and want[1][5] == 0


def test_strides(cuda_device):
    p, q, ids, u, nxt = case(5, 3, 1001, 5, cuda_device)
    big = torch.zeros(4, 5, 1203, device=cuda_device)
    big[:, :, 3:1004] = p.transpose(0, 1)
    pv = big[:, :, 3:1004].transpose(0, 1)  # rows of other strides, odd base
    qv = q.transpose(1, 2).contiguous().transpose(1, 2)  # inner stride
    iv = ids.t().contiguous().t()
    uv = torch.stack([u, u], dim=2)[:, :, 0]
    nv = torch.stack([nxt, nxt], dim=1)[:, 0]
    for args in ((pv, q, iv, uv, nv), (p, qv, ids, u, nxt)):
        tokens, accepted = verify_drafts(*args)
        want = verify(*on_host(p, q, ids, u, nxt))
        assert np.array_equal(tokens.cpu().numpy(), want[0])
        assert np.array_equal(accepted.cpu().numpy(), want[1])


@pytest.mark.parametrize("draft_given", [True, False])
def test_emitted_tokens_follow_the_target(cuda_device, draft_given):
    def run(*args):
        dev = [None if x is None else torch.from_numpy(np.ascontiguousarray(x)).to(cuda_device)
               for x in args]
        return on_host(*verify_drafts(*dev))

    got, p = emitted(draft_given, 64, run)
    assert np.abs(got - p).max() <= 2 / 64


@torch.inference_mode()  # as every capture among these tests: torch's generator state may be one of it
def test_two_graphs_and_eager_calls_share_nothing(cuda_device):
    """Two captured calls of other sizes, replayed in turn and at once on two streams, with eager
    calls between."""
    a = case(6, 4, 30000, 6, cuda_device)
    b = case(11, 2, 9000, 7, cuda_device)
    side = torch.cuda.Stream()
    verify_drafts(*a)
    graphs, outs = [], []
    for args in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(verify_drafts(*args))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for seed in range(4):
        for args, (s, k, v) in ((a, (6, 4, 30000)), (b, (11, 2, 9000))):
            for t, x in zip(args, case(s, k, v, 20 + seed, cuda_device)):
                t.copy_(x)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = verify_drafts(*a)
        torch.cuda.synchronize()
        for args, out in ((a, outs[0]), (b, outs[1]), (a, eager)):
            want = verify(*on_host(*args))
            assert np.array_equal(out[0].cpu().numpy(), want[0])
            assert np.array_equal(out[1].cpu().numpy(), want[1])
    stream = torch.cuda.current_stream().cuda_stream
    ws = _native._workspaces[(cuda_device.index or 0, stream, _native.WS_VERIFY)]
    assert ws[:16384 * 4].max() == 0


def test_refusals(cuda_device):
    p, q, ids, u, nxt = case(4, 3, 50, 8, cuda_device)
    for bad in ((p.half(), q, ids, u, nxt), (p, q[:, :2], ids, u, nxt), (p, q, ids.int(), u, nxt),
                (p, q, ids, u[:, :2], nxt), (p, q, ids, u, nxt.double()), (p, q, ids, u, nxt[:3]),
                (p, q.cpu(), ids, u, nxt), (p[:, :0], q[:, :0], ids, u, nxt),
                (p, q, ids, u, nxt, torch.zeros(4, device=cuda_device)),
                (p[..., :0], q[..., :0], ids, u, nxt)):
        with pytest.raises(AssertionError):
            verify_drafts(*bad)
    many = torch.zeros(1, 66, 10, device=cuda_device)
    with pytest.raises(_native.NativeLibraryError, match="64 drafts"):
        verify_drafts(many, None, torch.zeros(1, 65, dtype=torch.int64, device=cuda_device),
                      torch.zeros(1, 65, device=cuda_device), nxt[:1])
    tokens, accepted = verify_drafts(p[:0], q[:0], ids[:0], u[:0], nxt[:0])
    assert tokens.shape == (0, 4) and accepted.shape == (0,)


@pytest.mark.parametrize("vocab", [100, 9000, 600001])
@pytest.mark.parametrize("draft_given", [True, False])
def test_random_numbers_that_are_none(cuda_device, vocab, draft_given):
    """NaN: the draft is rejected, and the last index with a weight follows."""
    p, q, ids, u, nxt = case(6, 3, vocab, 9, cuda_device, off=0.3)
    q, nan = q if draft_given else None, float("nan")
    u = u * 0.01
    u[0, 0] = u[1, 2] = nan
    nxt[0] = nxt[2] = nan
    p[2, :, vocab * 2 // 3:] = 0.0
    p[3, :, vocab // 2:] = 0.0
    nxt[3] = 1.0
    want = check(p, q, ids, u, nxt)
    assert want[1][0] == 0 and want[1][1] <= 2
