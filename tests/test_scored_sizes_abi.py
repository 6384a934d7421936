"""Scales and caps whose scores fp32 does not hold in the exp2 domain are refused."""
from __future__ import annotations

import pytest

from engine.kernels import _native
from test_sampled_abi import _decode, _prefill


@pytest.mark.parametrize("call", [_decode, _prefill])
def test_sizes_past_the_largest(call):
    lib = _native.load()
    for name in ("scale", "softcap"):
        assert call(lib, **{name: 2.0 ** 127 * 1.0001}) == _native.PA_ERR_ARG
        assert f"{name} must be" in lib.pa_last_error().decode() and "2^127" in lib.pa_last_error().decode()
