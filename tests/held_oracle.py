"""Plain form of `place` with counts of held pages, on the CPU."""
from __future__ import annotations

from step_oracle import MOST


def place_held(table, starts, counts, tokens, page, free, taken, held):
    """(slots, positions, offsets, lengths, taken, held, table) as lists, token by
    token."""
    table = [list(row) for row in table]
    cols, taken = len(table[0]) if table else 0, max(0, taken)
    slots, positions, offsets, lengths, owned = [], [], [0], [], []
    for b, (s, n, own) in enumerate(zip(starts, counts, held)):
        s, n = max(0, s), min(max(0, n), tokens - len(slots))
        own = max(-(-s // page), own, 0)
        want = -(-min(s + n, cols * page) // page)
        got = own
        for col in range(own, want if n else own):
            there = taken < len(free)
            table[b][col] = free[taken] if there else -1
            taken, got = taken + 1, got + there
        for p in range(s, s + n):
            entry = table[b][p // page] if p // page < cols else -1
            slots.append(entry * page + p % page if entry >= 0 else -1)
            positions.append(min(p, MOST))
        offsets.append(len(slots))
        lengths.append(min(s + n, MOST))
        owned.append(min(got, MOST))
    spare = tokens - len(slots)
    return (slots + [-1] * spare, positions + [0] * spare, offsets, lengths,
            min(taken, MOST), owned, table)
