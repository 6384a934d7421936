"""Sampling from logits against the 64-bit oracle (needs an MI355X).

Tokens are whole numbers and have to be equal. Both sides weigh in 64 bits; they may differ
where u times the sum lies within 2^-44 per entry of a border, so numbers that near to one
(by the oracle) are refused as inputs before the kernel runs. Probabilities are rounded to
fp32 once: 2^-24 relative, and 2^-44 per entry of the sum.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from engine.kernels import _native
from engine.kernels.sampling import sample_tokens, sampling_probs
from oracle.sampling_oracle import probabilities, sample

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def rows_of(n, vocab, seed, device, dtype="fp16", spread=2.0):
    g = torch.Generator(device=device).manual_seed(seed)
    z = spread * torch.randn(n, vocab, generator=g, device=device)
    some = torch.randint(0, vocab, (n, 12), generator=g, device=device)
    z.scatter_(1, some, 6 + 4 * torch.rand(n, 12, generator=g, device=device))
    return z.to(TYPES[dtype]), torch.rand(n, generator=g, device=device)


def settings_of(row, **settings):
    return {k: (float(v[row]) if isinstance(v, torch.Tensor) else v) if k != "top_k" else
            int(v[row]) if isinstance(v, torch.Tensor) else v for k, v in settings.items()}


def check(z, u, **settings):
    """Tokens and probabilities of [rows, vocab] logits; the tokens."""
    # As the kernel sees them: numbers for all become fp32.
    settings = {k: v if isinstance(v, torch.Tensor) or k == "top_k" else float(np.float32(v))
                for k, v in settings.items()}
    host, numbers = z.double().cpu().numpy(), u.cpu().numpy()
    want, p = [], np.zeros_like(host)
    for r in range(len(host)):
        own = settings_of(r, **settings)
        token, gap = sample(host[r], numbers[r], **own)
        p[r] = probabilities(host[r], **own)
        # A number on a border (where sums are exact) is as good as one far from it.
        assert gap == 0 or gap > z.shape[1] * 2.0 ** -44, (r, gap)
        want.append(token)
    got = sample_tokens(z, u, **settings).cpu().numpy()
    assert np.array_equal(got, want), (got, want)
    probs = sampling_probs(z, **settings).cpu().double().numpy()
    assert np.array_equal(probs > 0, p >= 2.0 ** -149) or np.abs(probs - p).max() < 2.0 ** -120
    assert (np.abs(probs - p) <= p * (2.0 ** -24 + z.shape[1] * 2.0 ** -43) + 2.0 ** -149).all()
    return got


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("vocab", [1, 7, 8, 255, 256, 257, 1000, 1024, 1025, 4097, 32000, 100003,
                                   151936])
def test_matches_oracle(cuda_device, vocab, dtype):
    z, u = rows_of(3, vocab, vocab, cuda_device, dtype)
    check(z, u)
    check(z, u, temperature=0.0)
    check(z, u, temperature=0.7, top_k=20, top_p=0.8)
    check(z, u, temperature=1.4, top_p=0.95)
    check(z, u, min_p=0.05)
    check(z, u, temperature=0.8, top_k=50, top_p=0.9, min_p=0.1)


def test_settings_of_each_sequence(cuda_device):
    n = 40
    z, u = rows_of(n, 20011, 1, cuda_device)
    dev = cuda_device
    t = torch.tensor([0.0, 0.7, 1.0, 1.5, -1.0] * 8, device=dev)
    k = torch.tensor([0, 1, 40, 400, 20011, -3, 20010, 5000] * 5, dtype=torch.int32, device=dev)
    p = torch.tensor([1.0, 0.9, 0.5, 0.0, 2.0, 0.99, float("nan"), -1.0] * 5, device=dev)
    m = torch.tensor([0.0, 0.1, 0.0, 0.02, float("nan"), 3.0, -1.0, 1.0, 0.0, 0.3] * 4, device=dev)
    check(z, u, temperature=t, top_k=k, top_p=p, min_p=m)
    check(z, u, temperature=t, top_k=7, top_p=p, min_p=0.01)
    check(z, u, temperature=0.9, top_k=k, top_p=0.95, min_p=m)


@pytest.mark.parametrize("k", [2, 256, 257, 300, 1187, 1188, 1500, 2048, 2049, 5000, 60000, 151935])
def test_long_lists(cuda_device, k):
    """Beginnings that are ranked, radix-selected and narrowed by intervals, alone and with top-p."""
    z, u = rows_of(2, 151936, k, cuda_device, "fp32")
    check(z, u, temperature=1.2, top_k=k)
    check(z, u, temperature=1.2, top_k=k, top_p=0.9)
    check(z, u, temperature=2.0, top_k=k, top_p=0.99, min_p=0.001)


@pytest.mark.parametrize("p", [1e-6, 0.3, 0.9, 0.99, 0.9999, 1 - 2.0 ** -24])
@pytest.mark.parametrize("spread,t", [(0.01, 1.0), (2.0, 1.5), (5.0, 1.0), (2.0, 100.0), (2.0, 0.05)])
def test_nuclei(cuda_device, p, spread, t):
    for dtype in ("fp16", "fp32"):
        z, u = rows_of(2, 60000, int(p * 1000), cuda_device, dtype, spread)
        check(z, u, temperature=t, top_p=p)
        check(z, u, temperature=t, top_p=p, min_p=0.003)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("vocab", [300, 5000, 150000])
def test_equal_logits(cuda_device, vocab, dtype):
    """Rows of one value and of few: ties are cut by their index."""
    g = torch.Generator(device=cuda_device).manual_seed(3)
    u = torch.tensor([0.25, 0.5 + 2.0 ** -20, 0.75, 0.3], device=cuda_device)
    z = torch.zeros(4, vocab, device=cuda_device, dtype=TYPES[dtype])
    for settings in ({}, {"top_k": 100}, {"top_k": 299}, {"top_p": 0.5}, {"top_k": 250, "top_p": 0.5},
                     {"min_p": 0.5}, {"temperature": 0.0}, {"temperature": 1e-30, "top_k": 7}):
        got = check(z, u, **settings)
        if settings == {}:
            assert got[0] == vocab // 4
    z = torch.randint(-3, 4, (4, vocab), generator=g, device=cuda_device).to(TYPES[dtype])
    z[1] = -z[1].abs()  # zeros of both signs
    for settings in ({"top_k": 100}, {"top_k": vocab // 3}, {"top_p": 0.4}, {"top_p": 0.9, "top_k": 290},
                     {"temperature": 0.0}, {"temperature": 0.5, "min_p": 0.13}, {}):
        check(z, u, **settings)


def test_masked_and_odd_logits(cuda_device):
    """-inf, NaN and +inf among the logits, rows of nothing else, the type's lowest value."""
    inf, nan = float("inf"), float("nan")
    z, u = rows_of(12, 9001, 5, cuda_device, "fp16")
    z[0] = -inf
    z[1] = nan
    z[2, ::2] = nan
    z[3, 1:] = -inf
    z[4, 77] = inf
    z[5, [5, 9000]] = inf
    z[6] = torch.finfo(torch.float16).min
    z[7, :-1] = torch.finfo(torch.float16).min
    z[8] = inf
    z[9, 100:] = -inf
    z[10] = torch.finfo(torch.float16).max
    z[11, :5000] = -inf
    for settings in ({}, {"top_k": 3}, {"top_p": 0.9}, {"min_p": 0.1}, {"temperature": 0.0},
                     {"temperature": 0.01, "top_k": 500, "top_p": 0.999}, {"top_k": 8999},
                     {"temperature": inf, "top_p": 0.6}, {"temperature": inf}):
        got = check(z, u, **settings)
        assert got[0] == 0 and got[1] == 0 and got[3] == 0 and got[4] == 77
    assert (sampling_probs(z)[:2] == 0).all()


def test_border_numbers(cuda_device):
    """u of 0, the largest below 1, 1, above, negative and NaN."""
    for vocab in (200, 3001, 70000):
        z, _ = rows_of(1, vocab, 6, cuda_device, "fp32")
        for x in (0.0, 1.0, 7.5, -1.0, float("nan")):
            u = torch.full((1,), x, device=cuda_device)
            for settings in ({"top_k": 40}, {"top_p": 0.999}, {}):
                want = sample(z[0].double().cpu().numpy(), x, **{k: float(np.float32(v)) if k != "top_k"
                                                               else v for k, v in settings.items()})[0]
                assert int(sample_tokens(z, u, **settings)) == want, (vocab, x, settings)


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
def test_rows_of_sequences_and_strides(cuda_device, dtype):
    n, rows, vocab = 5, 3, 10007
    z, u = rows_of(n * rows, vocab, 7, cuda_device, dtype)
    k = torch.tensor([5, 0, 50, 3, 1000], dtype=torch.int32, device=cuda_device)
    want = check(z, u, temperature=0.9, top_k=k.repeat_interleave(rows), top_p=0.9)
    z3, u2 = z.view(n, rows, vocab), u.view(n, rows)
    big = torch.zeros(rows, n, vocab + 9, dtype=z.dtype, device=cuda_device)
    big[:, :, 3:-6] = z3.transpose(0, 1)
    wide = torch.stack([z3, z3], dim=3)[..., 0]  # inner stride
    uv = u2.t().contiguous().t()
    kv = torch.stack([k, k], dim=1)[:, 0]
    for zz in (z3, big[:, :, 3:-6].transpose(0, 1), wide):
        for uu, kk in ((u2, k), (uv, kv)):
            got = sample_tokens(zz, uu, 0.9, kk, 0.9)
            assert got.shape == (n, rows) and np.array_equal(got.cpu().numpy().reshape(-1), want)
            assert torch.equal(sampling_probs(zz, 0.9, kk, 0.9), sampling_probs(z3, 0.9, k, 0.9))


def test_many_rows(cuda_device):
    for n, vocab in ((3000, 301), (700, 3000), (16384, 40)):
        z, u = rows_of(n, vocab, n, cuda_device)
        got = sample_tokens(z, u, 0.8, 10, 0.9)
        pick = list(range(0, n, max(1, n // 50)))
        assert got[pick].tolist() == check(z[pick], u[pick], temperature=0.8, top_k=10, top_p=0.9).tolist()
    with pytest.raises(_native.NativeLibraryError, match="at most 16384 rows"):
        sample_tokens(torch.zeros(16385, 8, device=cuda_device), torch.zeros(16385, device=cuda_device))
    with pytest.raises(_native.NativeLibraryError, match="at most"):
        sampling_probs(torch.zeros(1, 2 ** 19 + 1, device=cuda_device))


def test_largest_vocabulary(cuda_device):
    z, u = rows_of(2, 2 ** 19, 8, cuda_device, "fp32")
    for settings in ({}, {"top_k": 3000}, {"temperature": 3.0, "top_p": 0.99}, {"top_k": 4097}):
        check(z, u, **settings)


def test_empty_and_repeated(cuda_device):
    none = sample_tokens(torch.zeros(0, 50, device=cuda_device), torch.zeros(0, device=cuda_device))
    assert none.shape == (0,) and none.dtype == torch.int64
    assert sampling_probs(torch.zeros(4, 0, 50, device=cuda_device)).shape == (4, 0, 50)
    z, u = rows_of(64, 50000, 9, cuda_device)
    a = (sample_tokens(z, u, 1.3, 0, 0.95), sampling_probs(z, 1.3, 0, 0.95))
    for _ in range(3):
        assert torch.equal(sample_tokens(z, u, 1.3, 0, 0.95), a[0])
        assert torch.equal(sampling_probs(z, 1.3, 0, 0.95), a[1])


def test_captured_and_on_another_stream(cuda_device):
    with torch.inference_mode():
        z, u = rows_of(9, 30011, 10, cuda_device)
        k = torch.tensor([5, 0, 1000] * 3, dtype=torch.int32, device=cuda_device)
        sample_tokens(z, u, 0.9, k, 0.9)
        torch.cuda.synchronize()
        graphs = []
        for _ in range(2):  # two graphs and eager calls share no workspace
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = sample_tokens(z, u, 0.9, k, 0.9), sampling_probs(z, 0.9, k, 0.9)
            graphs.append((graph, out))
        side = torch.cuda.Stream()
        for i in range(4):
            z2, u2 = rows_of(9, 30011, 20 + i, cuda_device)
            z.copy_(z2)
            u.copy_(u2)
            want = sample_tokens(z2, u2, 0.9, k, 0.9), sampling_probs(z2, 0.9, k, 0.9)
            for graph, out in graphs:
                graph.replay()
            torch.cuda.synchronize()
            for _, out in graphs:
                assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                got = sample_tokens(z2, u2, 0.9, k, 0.9)
            torch.cuda.current_stream().wait_stream(side)
            assert torch.equal(got, want[0])


def test_refusals(cuda_device):
    z, u = rows_of(2, 100, 11, cuda_device)
    for bad in (lambda: sample_tokens(z.double(), u), lambda: sample_tokens(z, u.double()),
                lambda: sample_tokens(z, u[:1]), lambda: sample_tokens(z[0], u[0]),
                lambda: sample_tokens(z, u, torch.ones(3, device=cuda_device)),
                lambda: sample_tokens(z, u, 1.0, torch.ones(2, device=cuda_device)),
                lambda: sample_tokens(z, u, 1.0, 2.5), lambda: sample_tokens(z.cpu(), u),
                lambda: sample_tokens(z, u.cpu()), lambda: sampling_probs(z, torch.ones(2)),
                lambda: sampling_probs(z[:, :0])):
        with pytest.raises(AssertionError):
            bad()
