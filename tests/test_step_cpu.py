"""CPU tests of the operators of a step of many tokens: what the C entry points
refuse (the pointers here are never followed), and the test oracle."""
from __future__ import annotations

import ctypes

import pytest

from cudalab_amd import _capi
from step_oracle import place
from test_attention_cpu import BAD_CACHE, P, _cache

BAD = _capi.CQ_ERR_INVALID_ARG


def _place(**change):
    a = _capi.CqPlace(
        starts=P[0], counts=P[1], free_pages=P[2], taken_in=P[3], table=P[4], slots=P[5],
        positions=P[6], offsets=P[7], lengths=P[8], taken_out=P[9], table_stride=7, tokens=100,
        free_count=50, table_cols=5, batch=3, page_size=16)
    for n, v in change.items():
        setattr(a, n, v)
    return _capi.load().cq_place(ctypes.byref(a), None)


@pytest.mark.parametrize("change", [
    dict(batch=0), dict(batch=-1), dict(batch=2 ** 31 - 1), dict(tokens=-1), dict(tokens=2 ** 31),
    dict(page_size=8), dict(page_size=48), dict(page_size=512), dict(free_count=-1),
    dict(free_pages=None), dict(table=None), dict(table=P[4] + 2), dict(table_cols=0),
    dict(table_stride=4), dict(table_cols=2 ** 27, table_stride=2 ** 27),
    *(dict([(n, None)]) for n in ("starts", "counts", "offsets", "lengths", "taken_out", "slots",
                                  "positions")),
    *(dict([(n, P[12] + 2)]) for n in ("starts", "counts", "free_pages", "taken_in", "positions",
                                       "offsets", "lengths", "taken_out")),
    dict(slots=P[5] + 4), dict(taken_out=P[3]), dict(lengths=P[0]), dict(offsets=P[8] - 12),
    dict(positions=P[5] + 796), dict(table=P[0]), dict(free_pages=P[4] + 64),
    dict(counts=P[4] - 4, taken_in=P[4] + 72)])
def test_place_refuses(change):
    assert _place(**change) == BAD
    assert _capi.last_error()
    assert _capi.load().cq_place(None, None) == BAD


def _rows(cache=None, dtype=0, tokens=9, slots=P[5], k=P[6], v=P[7], strides=(256, 128, 256, 128)):
    c = cache or _cache()
    return _capi.load().cq_kv_append_rows(ctypes.byref(c), dtype, tokens, slots, k, strides[0],
                                          strides[1], v, strides[2], strides[3], None)


def test_append_rows_refuses():
    for change in BAD_CACHE:
        assert _rows(_cache(**change)) == BAD, change
    for change in (dict(dtype=3), dict(tokens=0), dict(tokens=-1), dict(tokens=2 ** 31),
                   dict(slots=None), dict(k=None), dict(v=None), dict(k=P[6] + 1),
                   dict(slots=P[5] + 4), dict(k=P[0]), dict(v=P[1] + 64), dict(slots=P[2]),
                   dict(strides=(-1, 128, 256, 128)), dict(strides=(256, 128, 256, 2 ** 41))):
        assert _rows(**change) == BAD, change
    # more workgroups than a launch holds
    assert _rows(_cache(heads=65535), tokens=2 ** 20) == BAD
    assert _capi.load().cq_kv_append_rows(None, 0, 1, P[5], P[6], 1, 1, P[7], 1, 1, None) == BAD


def test_place_by_hand():
    """Two sequences of 16-token pages: one of 15 tokens gets two, one of none
    gets three, of which the list holds two."""
    got = place([[4, 9, 9], [9, 9, 9]], [15, 0], [3, 18], 23, 16, [7, 5])
    assert got[0][:3] == [4 * 16 + 15, 7 * 16, 7 * 16 + 1]
    assert got[0][3:19] == [5 * 16 + i for i in range(16)]
    assert got[0][19:] == [-1] * 4
    assert got[1] == [15, 16, 17, *range(18), 0, 0]
    assert got[2:5] == ([0, 3, 21], [18, 18], 3)
    assert got[5] == [[4, 7, 9], [5, -1, 9]]
