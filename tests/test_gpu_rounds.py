"""GPU tests of many rounds of drafts: checked, a few of them kept, checked again,
until the sequences are as long as their room."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from attention_oracle import assert_close, quantize
from conftest import announce
from test_gpu_decode_context import _pages_of
from test_gpu_prompt_model import _counts, _model, _x
from test_gpu_tree import tree_attention

pytestmark = pytest.mark.gpu
PAGE = 64


class _Watch:
    """What a model's calls of `place` and `forward` gave."""

    def __init__(self, m):
        self.m, self.placed, self.seen = m, None, []

    def __enter__(self):
        att = self.m.att
        place, forward = att.place, att.forward

        def placed(*a, **k):
            self.placed = place(*a, **k)
            return self.placed

        def attended(q, *a, **k):
            self.seen.append((q, forward(q, *a, **k)))
            return self.seen[-1][1]

        att.place, att.forward = placed, attended
        return self

    def __exit__(self, *exc):
        del self.m.att.place, self.m.att.forward


def _owned(table, lengths):
    return [e for row, n in zip(table, lengths) for e in row[:-(-n // PAGE)]]


@pytest.mark.parametrize("bits", [8, 4])
def test_rounds_until_the_room_is_full(cuda, bits):
    """Few drafts of each round are kept, so that many rounds begin ahead of a page
    that an earlier round took; some rounds keep nothing, and some are not followed
    by `accept`.  Every draft has a slot, no page is in two places, what is kept
    stays in the cache, and attention is the plain form's."""
    from cudalab_amd.prompt import chains
    T, lens, room = 16, [60, 37], 150
    tree, depth = chains(2, T, 2)
    see = np.unpackbits(tree.cpu().numpy().view(np.uint8), axis=-1,
                        bitorder="little")[..., :T].astype(bool)
    m = _model(2, room, bits, layers=1)
    pages = m.free.numel()
    announce(f"rounds of drafts, {bits} bits")
    kept = [[[], []] for _ in lens]                # of each sequence: rows of k, of v
    prompt_lens = list(lens)
    m.prompt(_x(sum(lens), 1024, seed=20), _counts(lens))
    r = 0
    while max(lens) + T <= room:
        announce(f"round {r}, lengths {lens}")
        with _Watch(m) as w:
            m.check(_x(2, T, 1024, seed=100 + r), tree, depth)
        slots, table = w.placed.slots.tolist(), m.table.tolist()
        assert min(slots) >= 0, (r, lens)
        assert len(set(slots)) == len(slots), (r, lens)
        owned = _owned(table, [n + T for n in lens])
        assert all(0 <= e < pages for e in owned) and len(set(owned)) == len(owned), (r, lens)
        assert m.taken.item() <= pages
        if r % 5 == 0 or 48 < lens[0] < 68 and r % 2:
            (q, out), = w.seen
            want, tol = tree_attention(q.cpu(), _pages_of(m.caches[0]), table,
                                       [n + T for n in lens], see)
            assert_close(out, want, tol, f"round {r}")
        r += 1
        if r % 7 == 3:                             # given up: the same place once more
            continue
        keep = torch.zeros(2, T, dtype=torch.bool, device="cuda")
        take = [r % 2, 3 * (r % 4 != 0)]
        for b, n in enumerate(take):
            keep[b, b:2 * n:2] = True              # of one chain
        (k, v), = m.drafts
        for b in range(2):
            at = keep[b].nonzero()[:, 0]
            for which, x in ((0, k), (1, v)):
                kept[b][which].append(x.view(2, T, -1, 128)[b, at].cpu())
        m.accept(keep)
        lens = [n + t for n, t in zip(lens, take)]
        assert m.lengths.tolist() == lens
    host, table = _pages_of(m.caches[0]), m.table.tolist()
    for b, n in enumerate(lens):
        for which in (0, 1):
            codes, scale = quantize(torch.cat(kept[b][which]).float().numpy(), bits)
            got, there = host.values(table[b], prompt_lens[b], len(codes), which)
            exact = codes.astype(np.float64) * scale.astype(np.float64)[..., None]
            assert there.all() and np.array_equal(got, exact.swapaxes(0, 1))
            assert len(codes) == n - prompt_lens[b]


@pytest.mark.parametrize("room,n", [(128, 120), (120, 110), (128, 128), (100, 99)])
def test_kept_drafts_past_the_room(cuda, room, n):
    """Kept drafts that the room has no place for are dropped: the tokens before them
    stay as they are, and the lengths count what is in the caches."""
    from cudalab_amd.prompt import chains
    T = 16
    m = _model(2, room, layers=1)
    announce(f"drafts past a room of {room}")
    m.prompt(_x(n + 30, 1024, seed=30), _counts([n, 30]))
    before = _pages_of(m.caches[0])
    m.check(_x(2, T, 1024, seed=31), *chains(2, T, 1))
    m.accept(torch.ones(2, T, dtype=torch.bool, device="cuda"))
    assert m.lengths.tolist() == [room, 30 + T]
    after, table = _pages_of(m.caches[0]), m.table.tolist()
    (k, v), = m.drafts
    for which, x in ((0, k), (1, v)):
        for b, (had, has) in enumerate(((n, room), (30, 30 + T))):
            old, _ = before.values(table[b], 0, had, which)
            got, there = after.values(table[b], 0, has, which)
            assert there.all() and np.array_equal(got[:, :had], old)
            codes, scale = quantize(x.view(2, T, -1, 128)[b, :has - had].cpu().float().numpy(), 8)
            exact = codes.astype(np.float64) * scale.astype(np.float64)[..., None]
            assert np.array_equal(got[:, had:], exact.swapaxes(0, 1))
