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


def prompt(q, k, v, offsets, k_offsets=None, causal=True, scale=None):
    """(out, tolerance) in FP64 of packed q (tokens, Hq, D) over k, v (keys, H, D),
    tensors on the CPU; sequence by sequence, row by row where V is not finite.

    Tolerance: the weights, rounded to the type (half a unit of each, or half the
    smallest spacing of fp16), the FP32 scores (D products and sums, then 8 more
    steps, of the sum of magnitudes) and exponentials, sums of m terms in FP32,
    and one rounding to the type."""
    import numpy as np

    from attention_oracle import SMALL, UNIT
    tokens, hq, D = q.shape
    g = hq // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out, tol = np.zeros((tokens, hq, D)), np.zeros((tokens, hq, D))
    qd, kd, vd = (x.double().numpy() for x in (q, k, v))
    k_offsets = offsets if k_offsets is None else k_offsets
    for b in range(len(offsets) - 1):
        at, n = offsets[b], offsets[b + 1] - offsets[b]
        kat, m = k_offsets[b], k_offsets[b + 1] - k_offsets[b]
        if n <= 0 or m <= 0:
            continue
        sees = np.ones((n, m), bool)
        if causal:
            sees = np.arange(m)[None] <= (m - n + np.arange(n))[:, None]
        some = sees.any(1)
        for h in range(hq):
            qq, kk, vv = qd[at:at + n, h], kd[kat:kat + m, h // g], vd[kat:kat + m, h // g]
            with np.errstate(all="ignore"):
                s = np.where(sees, qq @ kk.T * scale, -np.inf)
                size = np.where(sees, np.abs(qq) @ np.abs(kk).T * abs(scale), 0).max(1)
                top = s.max(1, keepdims=True)
                e = np.where(sees, np.exp(s - np.where(some[:, None], top, 0)), 0)
                p = e / np.where(some[:, None], e.sum(1, keepdims=True), 1)
                if np.isfinite(vv).all():
                    o, mag = p @ vv, p @ np.abs(vv)
                else:
                    o = np.stack([(p[i, sees[i], None] * vv[sees[i]]).sum(0) for i in range(n)])
                    fin = np.where(np.isfinite(vv), vv, 0)
                    mag = p @ np.abs(fin)
                err = 2 * (D + 8) * 2.0 ** -24 * (size + 8)
                t = (UNIT[q.dtype] + 2 * err[:, None] + (m + 8) * 2.0 ** -24) * mag
                if UNIT[q.dtype] == 2.0 ** -11:
                    t += m * 2.0 ** -24 * np.abs(np.where(np.isfinite(vv), vv, 0)).max()
                t += UNIT[q.dtype] * np.abs(o) + SMALL[q.dtype]
            out[at:at + n, h] = np.where(some[:, None], o, 0)
            tol[at:at + n, h] = t
    return out, tol
