"""The 8-bit pool's calls and the drafts' verification through the native call path and without
it: the same results, and the Python path for what is not a plain call (needs an MI355X)."""
from __future__ import annotations

import pytest
import torch

from _fp8_pool import Fp8Pool, int32, starts_of
from engine.kernels import _native
from engine.kernels import quantized_cache as qc
from engine.kernels.speculative import verify_drafts

pytestmark = pytest.mark.gpu


class Wrapped(torch.Tensor):
    """A tensor subclass: never a plain call."""


def calls(device, wrap=lambda t: t):
    """Every entry point once, on the same data: a list of output tensors."""
    pool = Fp8Pool([40, 2100, 7], 2, 64, 16, seed=1, device=device)
    g = torch.Generator().manual_seed(2)
    new = [5, 30, 7]
    starts = int32(starts_of(new), device)
    rows = [torch.randn(42, 2, 64, generator=g).half().to(device) for _ in range(2)]
    q = torch.randn(42, 14, 64, generator=g).half().to(device)
    args = [wrap(t) for t in pool.args()]
    qc.paged_kv_write_fp8(wrap(rows[0]), rows[1], *args, starts)
    qc.paged_kv_write_fp8(wrap(rows[0][:3]), rows[1][:3], *args)
    out = [pool.dk.view(torch.uint8), pool.dv.view(torch.uint8), pool.dks, pool.dvs]
    out += qc.paged_kv_read_fp8(*args, starts, 42)
    out.append(qc.paged_attention_decode_fp8(wrap(q[:3]), *args, 0.125))
    out.append(qc.paged_attention_prefill_fp8(wrap(q), *args, starts, 30, 0.125))
    out.append(qc.paged_attention_prefill_fp8(wrap(q[:12]), *args, int32([0, 4, 8, 12], device), 4, 0.125))
    p = torch.softmax(torch.randn(3, 4, 700, generator=g), dim=-1).to(device)
    d = torch.softmax(torch.randn(3, 3, 700, generator=g), dim=-1).to(device)
    ids = torch.randint(0, 700, (3, 3), generator=g).to(device)
    u, nxt = torch.rand(3, 3, generator=g).to(device), torch.rand(3, generator=g).to(device)
    for draft, counts in ((d, None), (None, int32([3, 0, 1], device))):
        out += verify_drafts(wrap(p), draft, ids, u, nxt, counts)
    return [t.as_subclass(torch.Tensor).clone() for t in out]


def same(a, b):
    assert len(a) == len(b)
    for x, y in zip(a, b):
        assert x.dtype == y.dtype and torch.equal(x, y)


def test_both_paths_give_the_same(cuda_device, monkeypatch):
    calls(cuda_device)  # the workspaces exist
    native = {"direct_call": 0, "direct_counted": 0}

    def counting(name):
        inner = getattr(_native, name)

        def call(*args):
            out = inner(*args)
            native[name] += out is not None
            return out
        return call

    with monkeypatch.context() as m:
        for name in native:
            m.setattr(_native, name, counting(name))
        direct = calls(cuda_device)
    assert native == {"direct_call": 3, "direct_counted": 5}, native
    for name in native:
        monkeypatch.setattr(_native, name, lambda *a: None)
    same(direct, calls(cuda_device))


def test_subclasses_take_the_python_path(cuda_device, monkeypatch):
    plain = calls(cuda_device)
    for name in ("direct_call", "direct_counted"):
        inner = getattr(_native, name)

        def refused(*args, inner=inner):
            out = inner(*args)
            assert out is None
            return out
        monkeypatch.setattr(_native, name, refused)
    same(plain, calls(cuda_device, wrap=lambda t: t.as_subclass(Wrapped)))


def test_strided_lengths_and_starts(cuda_device):
    """Lengths, starts and counts that are views of other strides."""
    pool = Fp8Pool([40, 100], 2, 64, 16, seed=3, device=cuda_device)
    q = torch.randn(9, 14, 64, generator=torch.Generator().manual_seed(4)).half().to(cuda_device)
    starts = int32([0, 4, 9], cuda_device)
    twice = lambda t: torch.stack([t, t + 1000], dim=1)[:, 0]
    k, v, ks, vs, t, n = pool.args()
    want = qc.paged_attention_prefill_fp8(q, k, v, ks, vs, t, n, starts, 5, 0.125)
    got = qc.paged_attention_prefill_fp8(q, k, v, ks, vs, t, twice(n), twice(starts), 5, 0.125)
    assert torch.equal(want, got)
    want = qc.paged_kv_read_fp8(k, v, ks, vs, t, n, starts, 9)
    got = qc.paged_kv_read_fp8(k, v, ks, vs, t, twice(n), twice(starts), 9)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    assert torch.equal(qc.paged_attention_decode_fp8(q[:2], k, v, ks, vs, t, n, 0.125),
                       qc.paged_attention_decode_fp8(q[:2], k, v, ks, vs, t, twice(n), 0.125))
