"""GPU tests of the pages, slots and positions of a packed batch: every number
equal to the plain form's, the table's other entries as they were."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import announce
from step_oracle import MOST, place

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def att(cuda):
    from cudalab_amd.build import build
    return build("attention")


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _check(att, table, starts, counts, tokens, page, free, taken=None, stride=None):
    announce(f"place batch={len(table)} tokens={tokens} page={page} free={len(free)}")
    cols = len(table[0])
    wide = torch.full((len(table), stride or cols), 77, dtype=torch.int32, device="cuda")
    wide[:, :cols] = _ints(table)
    dev = wide[:, :cols]
    got = att.place(dev, _ints(starts), _ints(counts), tokens, page, _ints(free),
                    None if taken is None else _ints([taken]))
    want = place(table, starts, counts, tokens, page, free, taken or 0)
    for name, g, w in zip((*got._fields, "table"), (*got, dev), want):
        w = np.array(w, dtype=np.int64).reshape(g.shape)
        assert np.array_equal(g.cpu().numpy(), w), name
    assert bool((wide[:, cols:] == 77).all())
    return got


def _random(rng, batch, most, before, page, cols):
    starts = rng.integers(0, before + 1, batch).tolist()
    counts = rng.integers(0, most + 1, batch).tolist()
    total = batch * cols + 5
    order = rng.permutation(total).tolist()
    table = [order[b * cols:(b + 1) * cols] for b in range(batch)]
    return table, starts, counts, rng.permutation(total).tolist()


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("batch,most,before", [(1, 1, 0), (1, 700, 5), (3, 40, 300),
                                               (64, 33, 100), (255, 4, 70), (256, 1, 64),
                                               (257, 9, 0), (700, 3, 40), (5, 3000, 17)])
def test_against_the_plain_form(att, page, batch, most, before):
    rng = np.random.default_rng(batch * 1000 + page)
    cols = (most + before) // page + 2
    table, starts, counts, free = _random(rng, batch, most, before, page, cols)
    tokens = sum(counts) + int(rng.integers(0, 3)) * 100
    _check(att, table, starts, counts, tokens, page, free, stride=cols + 3)


@pytest.mark.parametrize("batch", [4, 300])
def test_odd_calls(att, batch):
    """Empty sequences and calls, negative numbers, lengths past the table and
    past 31 bits, a list that ends, entries that are no page, rows that the
    tokens do not fit."""
    rng = np.random.default_rng(batch)
    table, starts, counts, free = _random(rng, batch, 50, 60, 16, 9)
    total = sum(counts)
    _check(att, table, starts, [0] * batch, 0, 16, free)
    _check(att, table, starts, [0] * batch, 9, 16, free)
    _check(att, table, starts, counts, total, 16, [])
    _check(att, table, starts, counts, total, 16, free[:7])
    _check(att, table, starts, counts, total, 16, free, taken=11)
    _check(att, table, starts, counts, total, 16, free, taken=len(free) - 3)
    _check(att, table, starts, counts, total, 16, free, taken=MOST)
    _check(att, table, starts, counts, total, 16, free, taken=-5)
    _check(att, table, starts, counts, total // 2, 16, free)
    _check(att, table, starts, counts, 1, 16, free)
    odd = [-3 if b % 3 == 0 else n for b, n in enumerate(starts)]
    _check(att, table, odd, [-n if b % 4 == 1 else n for b, n in enumerate(counts)], total, 16,
           free)
    _check(att, table, [n + 130 for n in starts], counts, total, 16, free)
    _check(att, table, [MOST] * batch, counts, total, 16, free)
    _check(att, table, [MOST - 3] * batch, counts, total, 16, free)
    _check(att, table, starts, [MOST] * batch, 501, 16, free)
    bad = [[-1 - c if (b + c) % 2 else MOST for c in range(9)] for b in range(batch)]
    _check(att, bad, starts, counts, total, 16, free)


def test_a_step_after_a_step(att):
    """Prompts, then single tokens: `taken` runs on, no page is handed out twice."""
    page, batch, cols = 16, 37, 12
    free = _ints(np.random.default_rng(0).permutation(batch * cols).tolist())
    table = torch.full((batch, cols), -1, dtype=torch.int32, device="cuda")
    counts = [(7 * b) % 50 for b in range(batch)]
    announce("place, a step after a step")
    p = att.place(table, _ints([0] * batch), _ints(counts), sum(counts), page, free)
    for _ in range(40):
        p = att.place(table, p.lengths, _ints([1] * batch), batch, page, free, p.taken)
    torch.cuda.synchronize()
    assert p.lengths.tolist() == [n + 40 for n in counts]
    pages = table[table >= 0].tolist()
    assert len(set(pages)) == len(pages) == p.taken.item()
    assert len(pages) == sum(-(-(n + 40) // page) for n in counts)
    assert all(free[:len(pages)].tolist().count(x) == 1 for x in pages[:20])


def test_graph_replays_with_new_lengths(att):
    page, batch, cols, tokens = 32, 5, 8, 300
    rng = np.random.default_rng(3)
    table0, starts0, counts0, free = _random(rng, batch, 60, 90, page, cols)
    table, starts, counts = _ints(table0), _ints(starts0), _ints(counts0)
    dfree, taken = _ints(free), _ints([0])
    announce("place in a graph")
    att.place(table, starts, counts, tokens, page, dfree, taken)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        p = att.place(table, starts, counts, tokens, page, dfree, taken)
    for i in range(4):
        _, s, n, _ = _random(rng, batch, 60, 90, page, cols)
        for dev, host in ((table, table0), (starts, s), (counts, n), (taken, [3 * i])):
            dev.copy_(_ints(host))
        g.replay()
        torch.cuda.synchronize()
        want = place(table0, s, n, tokens, page, free, 3 * i)
        for x, w in zip((*p, table), want):
            assert x.cpu().tolist() == (w if isinstance(w, list) else [w])


def test_on_another_stream(att):
    table, starts, counts, free = _random(np.random.default_rng(9), 6, 90, 40, 64, 4)
    side = torch.cuda.Stream()
    args = _ints(table), _ints(starts), _ints(counts), sum(counts), 64, _ints(free)
    torch.cuda.synchronize()
    announce("place on another stream")
    with torch.cuda.stream(side):
        p = att.place(*args)
    side.synchronize()
    want = place(table, starts, counts, sum(counts), 64, free)
    assert p.slots.tolist() == want[0] and args[0].tolist() == want[5]


def test_no_sequences(att):
    none = torch.empty(0, 3, dtype=torch.int32, device="cuda")
    p = att.place(none, _ints([]), _ints([]), 4, 16, _ints([1]), _ints([2]))
    assert p.slots.tolist() == [-1] * 4 and p.positions.tolist() == [0] * 4
    assert p.offsets.tolist() == [0] and p.lengths.tolist() == [] and p.taken.tolist() == [2]


def test_refusals(att):
    good = dict(block_table=_ints([[0, 1], [2, 3]]), starts=_ints([0, 0]), counts=_ints([3, 4]),
                tokens=9, page_size=16, free_pages=_ints([5, 6]), taken=_ints([0]))
    att.place(**good)
    t = good["block_table"]
    for change in (dict(block_table=None), dict(block_table=t.long()), dict(block_table=t[0]),
                   dict(block_table=t.cpu()), dict(block_table=t.t()), dict(starts=_ints([0])),
                   dict(starts=_ints([0, 0]).long()), dict(counts=_ints([1, 2, 3])),
                   dict(counts=[1, 2]), dict(tokens=-1), dict(tokens=2 ** 31), dict(tokens=1.0),
                   dict(tokens=True), dict(page_size=48), dict(page_size=512), dict(page_size=0),
                   dict(free_pages=None), dict(free_pages=_ints([[5], [6]])),
                   dict(free_pages=_ints([5, 6, 7, 8])[::2]), dict(taken=0),
                   dict(taken=_ints([0, 1])), dict(starts=t.view(-1)[:2]),
                   dict(free_pages=t.view(-1)), dict(block_table=t[:1].expand(2, 2))):
        with pytest.raises(RuntimeError):
            att.place(**{**good, **change})
