"""CPU tests of the sizes that the calls around attention accept: products that
pass 64 bits are refused, not wrapped (the pointers here are never followed)."""
from __future__ import annotations

import pytest

from cudalab_amd import _capi
from test_attention_cpu import _append, _cache, _slots


@pytest.mark.parametrize("heads,batch,tokens", [
    (100, 2 ** 30 + 12345, 2 ** 31 - 20),       # wraps to below zero
    (65535, 2 ** 31 - 1, 2 ** 31 - 1),
    (2 ** 15, 2 ** 30, 2 ** 23 - 30),           # 2^64 to the unit: wraps to 0
    (2 ** 15, 2 ** 30, 2 ** 23 - 14)])          # and a little more
def test_append_refuses_workgroups_past_64_bits(heads, batch, tokens):
    st = _append(_cache(heads=heads), _slots(batch=batch, tokens=tokens), stride=0)
    assert st == _capi.CQ_ERR_INVALID_ARG
    assert "workgroups" in _capi.last_error()
