"""The 8-bit pool's entry points check their arguments on the host before any launch (no GPU)."""
from __future__ import annotations

import pytest
import torch

from engine.kernels import _native
from engine.kernels import quantized_cache as qc

S = _native.i64_array
POOL = S([2048, 128, 64, 1])


def _write(lib, key=16, kstr=POOL, starts=16, seqs=2, tokens=9, hkv=2, d=64, bs=16, blocks=10,
           width=4, lens=16):
    rows = S([128, 64, 1])
    return lib.pa_kv_write_fp8(key, rows, 16, rows, 16, kstr, 16, POOL, 16, S([2, 1]), 16,
                               S([2, 1]), 16, S([4, 1]), lens, starts, seqs, tokens, hkv, d, bs,
                               blocks, width, None)


def _read(lib, key=16, kstr=POOL, kout=S([128, 64, 1]), starts=16, seqs=2, tokens=9, hkv=2, d=64,
          bs=16, blocks=10, width=4):
    return lib.pa_kv_read_fp8(16, kstr, 16, POOL, 16, S([2, 1]), 16, S([2, 1]), 16, S([4, 1]), 16,
                              starts, key, kout, 16, S([128, 64, 1]), seqs, tokens, hkv, d, bs,
                              blocks, width, None)


@pytest.mark.parametrize("call", [_write, _read])
def test_cache_argument_errors(call):
    lib = _native.load()
    assert call(lib, key=0) == _native.PA_ERR_ARG
    assert b"null" in lib.pa_last_error()
    assert call(lib, kstr=S([2048, 128, 64, 2])) == _native.PA_ERR_ARG
    assert b"stride" in lib.pa_last_error()
    for bad in (dict(hkv=0), dict(d=0), dict(bs=0), dict(blocks=0), dict(width=0)):
        assert call(lib, **bad) == _native.PA_ERR_ARG, bad
        assert b"positive" in lib.pa_last_error()
    assert call(lib, seqs=-1) == _native.PA_ERR_ARG
    assert call(lib, tokens=-1) == _native.PA_ERR_ARG
    # Nothing to do: no launch, no pointer is touched.
    assert call(lib, key=0, tokens=0) == _native.PA_OK
    assert call(lib, key=0, seqs=0) == _native.PA_OK


def test_cache_argument_errors_of_each_call():
    lib = _native.load()
    assert _write(lib, starts=None) == _native.PA_ERR_ARG  # 9 rows of 2 sequences need starts
    assert b"query_start_loc" in lib.pa_last_error()
    assert _read(lib, starts=None) == _native.PA_ERR_ARG
    assert _read(lib, kout=S([128, 64, 2])) == _native.PA_ERR_ARG
    # More blocks than one launch takes is refused, not cut.
    assert _write(lib, seqs=2 ** 31 - 1, tokens=2 ** 31 - 1) == _native.PA_ERR_UNSUPPORTED


def test_python_calls_need_the_gpu():
    codes = torch.zeros(4, 16, 2, 64).to(torch.float8_e4m3fn)
    scale = torch.ones(4, 2)
    tables, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    pool = (codes, codes, scale, scale, tables, lens)
    rows = torch.zeros(1, 2, 64, dtype=torch.float16)
    with pytest.raises(AssertionError):
        qc.paged_kv_write_fp8(rows, rows, *pool)
    with pytest.raises(AssertionError):
        qc.paged_kv_read_fp8(*pool, torch.tensor([0, 1], dtype=torch.int32), 1)


def _decode(lib, q=16, k=16, out=16, kstr=POOL, qstr=S([896, 64, 1]), hq=14, hkv=2, d=64, bs=16,
            blocks=10, width=4, seqs=2, ws=0, nbytes=0):
    return lib.pa_decode_fp8(q, qstr, k, kstr, 16, POOL, 16, S([2, 1]), 16, S([2, 1]), 16,
                             S([4, 1]), 16, out, S([896, 64, 1]), seqs, hq, hkv, d, bs, blocks,
                             width, 0.125, ws, nbytes, None)


def test_decode_argument_errors():
    lib = _native.load()
    for bad in (dict(q=0), dict(out=0), dict(k=8), dict(hq=15), dict(hkv=0), dict(bs=0), dict(blocks=0),
                dict(width=0), dict(seqs=-1), dict(kstr=S([2048, 128, 72, 1])),
                dict(kstr=S([-2048, 128, 64, 1])), dict(kstr=S([2048, 128, 64, 2])),
                dict(qstr=S([900, 64, 1])), dict(qstr=S([896, 64, 2]))):
        assert _decode(lib, **bad) == _native.PA_ERR_ARG, bad
        assert lib.pa_last_error()
    for bad in (dict(d=48), dict(hq=34), dict(width=2 ** 27)):
        assert _decode(lib, **bad) == _native.PA_ERR_UNSUPPORTED, bad
    assert _decode(lib, width=4096) == _native.PA_ERR_WORKSPACE  # long tables are split
    assert _decode(lib, seqs=0, q=0) == _native.PA_OK
    assert lib.pa_decode_fp8_workspace_bytes(2, 14, 2, 48, 16, 4) == 0
    assert lib.pa_decode_fp8_workspace_bytes(1, 14, 2, 64, 16, 4096) > 65536


def _prefill(lib, q=16, k=16, ks=16, kstr=POOL, qstr=S([896, 64, 1]), starts=16, hq=14, d=64,
             width=4, seqs=2, tokens=9, longest=5, scale=0.125):
    return lib.pa_prefill_attention_fp8(q, qstr, k, kstr, 16, POOL, ks, S([2, 1]), 16, S([2, 1]), 16,
                                        S([4, 1]), 16, starts, longest, 16, S([896, 64, 1]), seqs,
                                        tokens, hq, 2, d, 16, 10, width, scale, None, 0, None)


def test_prefill_argument_errors():
    lib = _native.load()
    for bad in (dict(q=0), dict(ks=0), dict(k=8), dict(hq=15), dict(width=0), dict(starts=0),
                dict(kstr=S([2048, 128, 72, 1])), dict(kstr=S([2048, 128, 64, 2])),
                dict(qstr=S([900, 64, 1])), dict(scale=0.0), dict(scale=float("inf")),
                dict(longest=-1), dict(seqs=-1)):
        assert _prefill(lib, **bad) == _native.PA_ERR_ARG, bad
        assert lib.pa_last_error()
    assert _prefill(lib, d=48) == _native.PA_ERR_UNSUPPORTED
    assert _prefill(lib, hq=34) == _native.PA_ERR_UNSUPPORTED
    assert _prefill(lib, width=4096) == _native.PA_ERR_WORKSPACE
    assert _prefill(lib, q=0, tokens=0) == _native.PA_OK
