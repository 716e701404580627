"""Plain forms of the operators of a step of many tokens, on the CPU, and what
their tests share."""
from __future__ import annotations

MOST = 2 ** 31 - 1


def place(table, starts, counts, tokens, page, free, taken=0):
    """(slots, positions, offsets, lengths, taken, table) as lists, token by
    token."""
    table = [list(row) for row in table]
    cols, taken = len(table[0]) if table else 0, max(0, taken)
    slots, positions, offsets, lengths = [], [], [0], []
    for b, (s, n) in enumerate(zip(starts, counts)):
        s, n = max(0, s), min(max(0, n), tokens - len(slots))
        held = -(-s // page)
        want = -(-min(s + n, cols * page) // page)
        for col in range(held, want if n else held):
            table[b][col] = free[taken] if taken < len(free) else -1
            taken += 1
        for p in range(s, s + n):
            entry = table[b][p // page] if p // page < cols else -1
            slots.append(entry * page + p % page if entry >= 0 else -1)
            positions.append(min(p, MOST))
        offsets.append(len(slots))
        lengths.append(min(s + n, MOST))
    spare = tokens - len(slots)
    return (slots + [-1] * spare, positions + [0] * spare, offsets, lengths,
            min(taken, MOST), table)
