"""GPU tests of attention over the cache for tokens that form a tree, against the
plain form in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from attention_oracle import Pages, assert_close, attention
from conftest import announce

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def att(cuda):
    from cudalab_amd.build import build
    return build("attention")


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _bits(see):
    """see (B, T, T) truth values as int64 (B, T, words)."""
    B, T, _ = see.shape
    words = (T + 63) // 64
    wide = np.zeros((B, T, words * 64), bool)
    wide[..., :T] = see
    packed = np.packbits(wide, axis=-1, bitorder="little")
    return torch.from_numpy(packed.view("<i8").reshape(B, T, words).copy())


def tree_attention(q, pages, table, lengths, see, counts=None, prefix=None, scale=None):
    """(out, tolerance): each query alone, over a table of the very keys that it
    sees, by the plain form for a single token."""
    B, T, Hq, D = q.shape
    out, tol = np.zeros((B, T, Hq, D)), np.zeros((B, T, Hq, D))
    for b in range(B):
        n = T if counts is None else min(T, max(0, counts[b]))
        room = len(table[b]) * pages.page
        for t in range(n):
            first = lengths[b] - n
            places = [p for p in range(max(0, min(lengths[b], room)))
                      if p < first or see[b, t, p - first]]
            # single tokens in pages of one key: gathered codes and scales
            one = _Gathered(pages, table[b], places)
            o, e = attention(q[b:b + 1, t:t + 1], one, [list(range(len(one.k)))],
                             [len(one.k)], None, _shift(prefix, pages, one), scale)
            out[b, t], tol[b, t] = o[0, 0], e[0, 0]
    return out, tol


class _Gathered(Pages):
    """The keys at `places` of one sequence, a page each."""

    def __init__(self, pages, table, places):
        self.bits, self.page, self.dim, self.heads = pages.bits, 1, pages.dim, pages.heads
        at = [(table[p // pages.page], p % pages.page) for p in places]
        at = [(e, o) for e, o in at if 0 <= e < len(pages.k)]
        e, o = np.array([x[0] for x in at], int), np.array([x[1] for x in at], int)
        self.k = pages.k[e, :, o][:, :, None]
        self.v = pages.v[e, :, o][:, :, None]
        self.scales = pages.scales[e, :, :, o][..., None]
        self.all = pages


def _shift(prefix, pages, one):
    """The prefix's keys behind the gathered ones, as pages of one key."""
    if prefix is None:
        return None
    table, n = prefix
    more = _Gathered(pages, table, range(n))
    first = len(one.k)
    one.k, one.v = np.concatenate((one.k, more.k)), np.concatenate((one.v, more.v))
    one.scales = np.concatenate((one.scales, more.scales))
    return list(range(first, first + len(more.k))), len(more.k)


def _ancestors(B, T, rng):
    see = np.zeros((B, T, T), bool)
    for b in range(B):
        for t in range(T):
            up = int(rng.integers(-1, t)) if t else -1
            if up >= 0:
                see[b, t] = see[b, up]
            see[b, t, t] = True
    return see


def _case(B, T, hq, h, d, page, bits, dtype, lengths, seed=0):
    rng = np.random.default_rng(seed)
    cols = max(1, -(-max(lengths) // page))
    pages = Pages(B * cols + 2, h, d, page, bits, seed=seed)
    top = 127 if bits == 8 else 7
    pages.scales *= 1.7 / top
    order = rng.permutation(B * cols + 2).tolist()
    table = [order[b * cols:(b + 1) * cols] for b in range(B)]
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(B, T, hq, d, generator=g) * 1.5).to(DT[dtype])
    return rng, pages, table, q, order[B * cols:]


def _check(att, q, pages, table, lengths, see, counts=None, prefix=None, scale=None, what=""):
    announce(f"tree {what} {q.dtype} q {tuple(q.shape)} lengths {lengths} counts {counts}")
    pre = None if prefix is None else (_ints(prefix[0]), prefix[1])
    got = att.forward(q.cuda(), pages.device(), _ints(table), _ints(lengths),
                      None if counts is None else _ints(counts), prefix=pre, scale=scale,
                      tree=_bits(see).cuda())
    want, tol = tree_attention(q, pages, table, lengths, see, counts, prefix, scale)
    assert_close(got, want, tol, what)
    return got


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("d,hq,h,page,dtype", [(64, 7, 1, 32, "bf16"), (128, 8, 2, 64, "fp16"),
                                               (256, 4, 2, 16, "fp16"), (128, 2, 2, 128, "bf16")])
@pytest.mark.parametrize("T,lengths", [(1, [1, 130]), (2, [2, 1, 0]), (13, [13, 70, 5, 200]),
                                       (16, [64, 65, 80]), (33, [300, 33]), (64, [64, 150]),
                                       (70, [70, 133])])
def test_against_the_plain_form(att, bits, d, hq, h, page, dtype, T, lengths):
    """One to more than 64 tokens, sequences shorter than the tree, trees that
    begin and end anywhere in a tile."""
    rng, pages, table, q, _ = _case(len(lengths), T, hq, h, d, page, bits, dtype, lengths)
    _check(att, q, pages, table, lengths, _ancestors(len(lengths), T, rng))


@pytest.mark.parametrize("bits,T", [(8, 9), (4, 40), (8, 130)])
def test_counts_any_bits_and_a_prefix(att, bits, T):
    """Fewer tokens than the call's, bits that are no tree (none at all, later
    tokens, tokens past the count), a prefix."""
    lengths = [T + 3, 90, T, 0, 150]
    counts = [T, T // 2, 0, 3, T + 9]
    rng, pages, table, q, spare = _case(5, T, 6, 2, 128, 64, bits, "fp16", lengths, 3)
    see = rng.random((5, T, T)) < 0.3
    see[:, 1] = False
    see[0, 0] = True
    _check(att, q, pages, table, lengths, see, counts, what="any bits")
    _check(att, q, pages, table, lengths, see, counts, (spare, 100), 0.2, "prefix")
    got = att.forward(q.cuda(), pages.device(), _ints(table), _ints([T] * 5), None,
                      tree=torch.zeros_like(_bits(see)).cuda())
    assert bool((got == 0).all()), "rows that see nothing"


def test_a_chain_is_the_call_without_a_tree(att):
    """Each token under the one before it: bit for bit what causal order gives."""
    for T, lengths in ((5, [5, 77, 1501]), (40, [40, 64, 900])):
        rng, pages, table, q, _ = _case(3, T, 8, 1, 128, 64, 8, "bf16", lengths, 5)
        see = np.tril(np.ones((3, T, T), bool))
        announce(f"tree as a chain T={T}")
        args = q.cuda(), pages.device(), _ints(table), _ints(lengths)
        a, b = att.forward(*args, tree=_bits(see).cuda()), att.forward(*args)
        want, tol = attention(q, pages, table, lengths)
        assert_close(a, want, tol, "chain")
        assert_close(b, want, tol, "causal")


@pytest.mark.parametrize("T", [6, 48])
def test_what_is_not_seen_leaves_no_trace(att, T):
    """A branch whose keys have scales of NaN and Inf: only rows of that branch
    turn NaN; positions without a page are not seen."""
    lengths = [T + 100, T + 30]
    rng, pages, table, q, _ = _case(2, T, 4, 1, 64, 16, 8, "fp16", lengths, 7)
    see = _ancestors(2, T, rng)
    bad = 2
    for which, value in ((0, np.nan), (1, np.inf)):
        p = lengths[0] - T + bad
        pages.scales[table[0][p // 16], :, which, p % 16] = value
    table[1][0] = -1
    got = _check(att, q, pages, table, lengths, see, what="a bad branch").cpu()
    hit = torch.from_numpy(see[0][:, bad])
    assert bool(got[0][hit].isnan().all()) and bool(got[0][~hit].isfinite().all())


def test_long_contexts(att):
    rng, pages, table, q, _ = _case(2, 21, 8, 1, 128, 64, 4, "fp16", [5000, 777], 8)
    _check(att, q, pages, table, [5000, 777], _ancestors(2, 21, rng), what="long")


def test_graph_replays_with_new_trees(att):
    T, lengths = 12, [40, 200, 12]
    rng, pages, table, q, _ = _case(3, T, 8, 2, 64, 32, 8, "fp16", lengths, 9)
    cache, dq, tab, lens = pages.device(), q.cuda(), _ints(table), _ints(lengths)
    bits = _bits(_ancestors(3, T, rng)).cuda()
    out = torch.empty_like(dq)
    att.forward_into(dq, cache, tab, lens, out, tree=bits)
    torch.cuda.synchronize()
    announce("tree in a graph")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        att.forward_into(dq, cache, tab, lens, out, tree=bits)
    for new in ([40, 200, 12], [12, 13, 180], [5, 64, 100]):
        see = _ancestors(3, T, rng)
        bits.copy_(_bits(see))
        lens.copy_(_ints(new))
        g.replay()
        torch.cuda.synchronize()
        want, tol = tree_attention(q, pages, table, new, see)
        assert_close(out, want, tol, f"replay {new}")


def test_refusals(att):
    rng, pages, table, q, _ = _case(2, 5, 4, 2, 64, 16, 8, "fp16", [9, 30])
    good = dict(q=q.cuda(), cache=pages.device(), block_table=_ints(table),
                lengths=_ints([9, 30]), tree=_bits(_ancestors(2, 5, rng)).cuda())
    att.forward(**good)
    t = good["tree"]
    for bad in (t.int(), t[:1], t[:, :4], t[..., 0], t.cpu(), t.tolist(), 3,
                torch.cat((t, t), -1), torch.cat((t, t), -1)[..., :1]):
        with pytest.raises(RuntimeError):
            att.forward(**{**good, "tree": bad})
    out = torch.empty_like(good["q"])
    with pytest.raises(RuntimeError):
        att.forward_into(**good, out=t.view(torch.float16))
    flat = torch.zeros(out.numel() // 4, dtype=torch.int64, device="cuda")
    out = flat.view(torch.float16).view(out.shape)
    with pytest.raises(RuntimeError):
        att.forward_into(**{**good, "tree": flat[:10].view(2, 5, 1)}, out=out)
