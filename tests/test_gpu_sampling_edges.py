"""Sampling where single entries weigh less than the sums' unit, and past the rows that are
shared by workgroups, against the 64-bit oracle (needs an MI355X).

A token drawn has a weight of 2^-45 of the largest at least. Tokens have to be equal; inputs with
a weight within one part in 10^9 of that border are refused before the kernel runs.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from engine.kernels.sampling import sample_tokens
from oracle.sampling_oracle import kept_weights, sample
from test_gpu_sampling import check, rows_of

pytestmark = pytest.mark.gpu

BORDER = 2.0 ** -45


def check_ends(z, **settings):
    """Tokens at the ends of the numbers: 0, 1, above 1 and NaN."""
    settings = {k: v if k == "top_k" else float(np.float32(v)) for k, v in settings.items()}
    host = z.double().cpu().numpy()
    for row in host:
        w = kept_weights(row, **settings)
        assert (np.abs(w / BORDER - 1) > 1e-9).all()
    for x in (0.0, 1.0, 3.0, float("nan")):
        want = [sample(row, x, **settings)[0] for row in host]
        got = sample_tokens(z, torch.full((len(z),), x, device=z.device), **settings)
        assert got.tolist() == want, x


@pytest.mark.parametrize("vocab,k", [(151936, 400), (100003, 500), (60000, 3000)])
def test_low_temperatures_with_many_kept(cuda_device, vocab, k):
    z, _ = rows_of(60, vocab, k, cuda_device)
    check_ends(z, temperature=0.2, top_k=k)


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
@pytest.mark.parametrize("settings", [dict(top_k=45000), dict(min_p=1e-15), dict(top_k=45000, min_p=1e-15),
                                      dict(top_k=20000, top_p=0.999), dict()])
def test_pieces_of_entries_below_a_unit(cuda_device, settings, dtype):
    """The first and last thousands of a row hold only entries of 2^-45.9 to 2^-45.1 of the
    largest, some or all of them kept; the first and last index nothing."""
    vocab, top = 50000, 9.0
    g = torch.Generator(device=cuda_device).manual_seed(5)
    z = top - 31.1 * torch.rand(3, vocab, generator=g, device=cuda_device)
    for ends in (slice(0, 5000), slice(-5000, None)):
        z[:, ends] = top - 31.26 - 0.55 * torch.rand(3, 5000, generator=g, device=cuda_device)
    z[:, 0] = z[:, -1] = -float("inf")
    z[0, 25000], z[1, 24999], z[2, 30000] = top, top, top
    z = z.to({"fp16": torch.float16, "fp32": torch.float32}[dtype])
    check_ends(z, **settings)

def test_rows_past_those_that_are_shared(cuda_device):
    """Rows from 2048 on have no room to be shared in; long lists there take one workgroup each."""
    n, vocab = 2100, 4000
    z, u = rows_of(n, vocab, 12, cuda_device)
    pick = [0, 511, 512, 1000, 2046, 2047, 2048, 2049, 2099]
    for settings in (dict(temperature=5.0, top_p=0.97), dict(temperature=5.0, min_p=0.002),
                     dict(top_k=2500), dict(temperature=3.0, top_k=2500, top_p=0.95), dict(temperature=0.9)):
        got = sample_tokens(z, u, **settings)
        assert got[pick].tolist() == check(z[pick], u[pick], **settings).tolist(), settings
