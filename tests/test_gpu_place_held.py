"""GPU tests of `place` with counts of held pages: every number equal to the plain
form's, the table's other entries as they were."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import announce
from held_oracle import place_held
from step_oracle import MOST
from test_gpu_place import _ints, _random

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def att(cuda):
    from cudalab_amd.build import build
    return build("attention")


def _same(got, dev, want):
    for name, g, w in zip((*got._fields, "table"), (*got, dev), want, strict=True):
        w = np.array(w, dtype=np.int64).reshape(g.shape)
        assert np.array_equal(g.cpu().numpy(), w), name


def _check(att, table, starts, counts, tokens, page, free, held, taken=None):
    announce(f"place held batch={len(table)} tokens={tokens} page={page} free={len(free)}")
    cols = len(table[0])
    wide = torch.full((len(table), cols + 3), 77, dtype=torch.int32, device="cuda")
    wide[:, :cols] = _ints(table)
    dev, given = wide[:, :cols], _ints(held)
    got = att.place(dev, _ints(starts), _ints(counts), tokens, page, _ints(free),
                    None if taken is None else _ints([taken]), held=given)
    _same(got, dev, place_held(table, starts, counts, tokens, page, free, taken or 0, held))
    assert bool((wide[:, cols:] == 77).all()) and given.tolist() == held


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("batch,most,before", [(1, 1, 0), (1, 700, 5), (3, 40, 300), (64, 33, 100),
                                               (255, 4, 70), (256, 16, 64), (257, 9, 0),
                                               (700, 3, 40), (5, 3000, 17)])
def test_against_the_plain_form(att, page, batch, most, before):
    rng = np.random.default_rng(batch * 1000 + page)
    cols = (most + before) // page + 3
    table, starts, counts, free = _random(rng, batch, most, before, page, cols)
    held = rng.integers(0, cols + 1, batch).tolist()
    total = sum(counts)
    _check(att, table, starts, counts, total + 100, page, free, held)
    _check(att, table, starts, counts, total // 2, page, free, held, 3)
    _check(att, table, starts, counts, total, page, free[:len(free) // 3], held)
    _check(att, table, starts, counts, total, page, [], held)


@pytest.mark.parametrize("batch", [4, 300])
def test_odd_counts(att, batch):
    """Counts below zero, past the table and past 31 bits; entries that are no page;
    a list that ends inside a sequence, or ended before."""
    rng = np.random.default_rng(batch)
    table, starts, counts, free = _random(rng, batch, 50, 60, 16, 9)
    total = sum(counts)
    for held in ([-5] * batch, [MOST] * batch, [9] * batch, [-MOST - 1] * batch,
                 [(b * 7) % 11 - 1 for b in range(batch)]):
        _check(att, table, starts, counts, total, 16, free, held)
        _check(att, table, starts, [0] * batch, 9, 16, free, held)
        _check(att, table, [MOST - 3] * batch, counts, total, 16, free, held)
        _check(att, table, starts, counts, total, 16, free[:5], held)
        for taken in (11, len(free) - 3, MOST, -5):
            _check(att, table, starts, counts, total, 16, free, held, taken)
        bad = [[-1 - c if (b + c) % 2 else MOST for c in range(9)] for b in range(batch)]
        _check(att, bad, starts, counts, total, 16, free, held)


def test_graph_replays_with_new_counts(att):
    """A step whose lengths, taken and held go on from replay to replay (most sequences
    start with a page that the table does not have: their first tokens get no slot)."""
    page, batch, cols, T = 16, 5, 9, 6
    free = np.random.default_rng(1).permutation(batch * cols).tolist()
    host = [[-1] * cols for _ in range(batch)], [3 * b for b in range(batch)], 0, [0] * batch
    table, starts, taken, held = _ints(host[0]), _ints(host[1]), _ints([0]), _ints(host[3])
    counts, dfree = _ints([T] * batch), _ints(free)
    announce("place held in a graph")
    att.place(table.clone(), starts, counts, batch * T, page, dfree, taken, held=held)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        p = att.place(table, starts, counts, batch * T, page, dfree, taken, held=held)
        starts += 1                            # one of six drafts is kept
        taken.copy_(p.taken)
        held.copy_(p.held)
    tab, at, gone, own = host
    for i in range(20):
        g.replay()
        torch.cuda.synchronize()
        want = place_held(tab, at, [T] * batch, batch * T, page, free, gone, own)
        _same(p, table, want)
        tab, gone, own, at = want[6], want[4], want[5], [n + 1 for n in at]


def test_none_and_refusals(att):
    none = torch.empty(0, 3, dtype=torch.int32, device="cuda")
    p = att.place(none, _ints([]), _ints([]), 4, 16, _ints([1]), _ints([2]), held=_ints([]))
    assert p.slots.tolist() == [-1] * 4 and p.held.tolist() == [] and p.taken.tolist() == [2]
    good = dict(block_table=_ints([[0, 1], [2, 3]]), starts=_ints([0, 0]), counts=_ints([3, 4]),
                tokens=9, page_size=16, free_pages=_ints([5, 6]), held=_ints([1, 0]))
    p = att.place(**good)
    assert p.held.tolist() == [1, 1] and p.taken.tolist() == [1]
    assert good["block_table"].tolist() == [[0, 1], [5, 3]]
    t = good["block_table"]
    for held in (0, [1, 0], _ints([1]), _ints([1, 0]).long(), _ints([1, 0]).cpu(),
                 _ints([1, 0, 1, 0])[::2], t.view(-1)[:2], _ints([[1, 0]])):
        with pytest.raises(RuntimeError):
            att.place(**{**good, "held": held})
