"""CPU tests of `place` with counts of held pages: what the C entry refuses (the
pointers here are never followed), and the plain form over many rounds of drafts."""
from __future__ import annotations

import ctypes

import pytest

from cudalab_amd import _capi
from held_oracle import place_held
from step_oracle import place
from test_attention_cpu import P

BAD = _capi.CQ_ERR_INVALID_ARG


def _place(held_in=P[10], held_out=P[11], **change):
    a = _capi.CqPlace(
        starts=P[0], counts=P[1], free_pages=P[2], taken_in=P[3], table=P[4], slots=P[5],
        positions=P[6], offsets=P[7], lengths=P[8], taken_out=P[9], table_stride=7, tokens=100,
        free_count=50, table_cols=5, batch=3, page_size=16)
    for n, v in change.items():
        setattr(a, n, v)
    return _capi.load().cq_place_held(ctypes.byref(a), held_in, held_out, None)


@pytest.mark.parametrize("change", [
    dict(held_in=P[10] + 2), dict(held_out=P[11] + 1), dict(held_out=P[10]),
    dict(held_out=P[10] + 8), dict(held_out=P[0]), dict(held_in=P[8]), dict(held_in=P[4] + 72),
    dict(held_out=P[9] - 8), dict(held_out=P[5] + 796), dict(held_out=P[2] + 196),
    dict(held_in=P[9]), dict(batch=0), dict(tokens=-1), dict(page_size=24), dict(table=None),
    dict(table_stride=4), dict(lengths=P[0])])
def test_refusals(change):
    assert _place(**change) == BAD
    assert _capi.last_error()
    assert _capi.load().cq_place_held(None, None, None, None) == BAD


def test_by_hand():
    """16-token pages: a sequence of 15 tokens that owns two entries uses them before
    it takes one; one whose third page the list does not have holds two."""
    got = place_held([[4, 6, 9], [9, 9, 9]], [15, 0], [20, 33], 53, 16, [7, 5, 3], 0, [2, 0])
    assert got[0][:20] == [4 * 16 + 15, *(6 * 16 + i for i in range(16)),
                           *(7 * 16 + i for i in range(3))]
    assert got[0][20:] == [*(5 * 16 + i for i in range(16)), *(3 * 16 + i for i in range(16)), -1]
    assert got[4:6] == (4, [3, 2]) and got[6] == [[4, 6, 7], [5, 3, -1]]


def test_without_more_than_the_starts_need():
    args = [[4, 9, 9], [9, 9, 9]], [15, 0], [3, 18], 23, 16, [7, 5], 0
    got = place_held(*args, [1, -3])
    assert got[:5] + got[6:] == place(*args)


def test_rounds_of_drafts_lose_no_page():
    """One or two of 16 drafts kept each round, until the room is full: the counts
    of held pages keep every page with its sequence.  (With starts alone the list of
    as many pages as the tables hold ends in the second round.)"""
    page, cols, T = 64, 3, 16
    free = [3, 1, 5, 0, 4, 2]
    table, lens, taken, held = [[-1] * cols for _ in range(2)], [0, 0], 0, [0, 0]
    got = place_held(table, lens, [60, 37], 97, page, free, taken, held)
    lens, taken, held, table = got[3], got[4], got[5], got[6]
    plain = [list(r) for r in table], taken
    lost = None
    for r in range(40):
        got = place_held(table, lens, [T] * 2, 2 * T, page, free, taken, held)
        slots, taken, held, table = got[0], got[4], got[5], got[6]
        assert min(slots) >= 0 and len(set(slots)) == 2 * T
        assert taken <= len(free)
        pages = [e for row, n in zip(table, held) for e in row[:n]]
        assert len(set(pages)) == len(pages) == taken and min(pages) >= 0
        old = place(plain[0], lens, [T] * 2, 2 * T, page, free, plain[1])
        plain = old[5], old[4]
        if lost is None and min(old[0]) < 0:
            lost = r
        lens = [n + k for n, k in zip(lens, (1, r % 3))]
    assert lost is not None
