"""GPU tests of attention over the quantized cache against the formula in 64
bits: head groups, types, pages, lengths from nothing up, several new tokens,
shared prefixes, stale and missing pages."""
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


def _fill(pages, table, n, rng, peak=1.0):
    """Valid codes and scales of about unit values for a sequence's n tokens."""
    top = 127 if pages.bits == 8 else 7
    for i in range(n):
        p, off = table[i // pages.page], i % pages.page
        for which in (0, 1):
            codes = rng.integers(-top, top + 1, (pages.heads, pages.dim))
            pages.put(p, off, which, codes,
                      rng.uniform(0.5, 1.5, pages.heads) * peak * 1.7 / top)


def _setup(lens, heads, dim, page, bits, prefix=0, seed=0, stale="nan", peak=1.0):
    rng = np.random.default_rng(seed)
    need = [max(1, -(-n // page)) for n in lens]
    ahead = -(-prefix // page)
    order = rng.permutation(sum(need) + ahead + 1).tolist()
    pages = Pages(len(order), heads, dim, page, bits, seed, stale)
    ptable, order = order[:ahead], order[ahead:]
    _fill(pages, ptable, prefix, rng, peak)
    table = []
    for n, w in zip(lens, need):
        row, order = order[:w], order[w:]
        _fill(pages, row, n, rng, peak)
        table.append(row + [-1] * (max(need) - w))
    return pages, table, ptable


def _run(att, pages, table, lens, q, what, counts=None, prefix=None, scale=None):
    out = att.forward(q.cuda(), pages.device(), _ints(table), _ints(lens),
                      None if counts is None else _ints(counts),
                      prefix=None if prefix is None else (_ints(prefix[0]), prefix[1]),
                      scale=scale)
    assert out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous()
    want, tol = attention(q, pages, table, lens, counts, prefix, scale)
    assert_close(out, want, tol, what)
    return out


def _q(b, t, h, d, dtype, seed=0, by=1.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(b, t, h, d, generator=g) * by).to(DT[dtype])


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("dim,page,heads,group", [
    (128, 64, 2, 8), (64, 16, 3, 1), (256, 32, 1, 4), (128, 128, 1, 16), (64, 256, 2, 7),
    (128, 16, 1, 33), (256, 64, 2, 16), (64, 64, 1, 64)])
def test_one_token(att, bits, dtype, dim, page, heads, group):
    lens = [0, 1, 15, 16, 17, 63, 64, 65, 130, 300]
    pages, table, _ = _setup(lens, heads, dim, page, bits, seed=dim + page)
    announce(f"attention one token {bits} {dtype} d={dim} page={page} {heads}x{group}")
    out = _run(att, pages, table, lens, _q(len(lens), 1, heads * group, dim, dtype), "one token")
    assert bool((out[0] == 0).all())


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("tokens,group,dim", [(2, 8, 128), (5, 7, 64), (3, 1, 128), (17, 4, 64),
                                              (9, 2, 256), (40, 3, 128), (130, 1, 64)])
def test_several_tokens(att, bits, tokens, group, dim):
    """Causal among the new tokens; sequences shorter than them leave rows
    empty; ragged counts."""
    lens = [0, 1, tokens - 1, tokens, tokens + 1, 64, 200]
    counts = [0, 1, tokens, tokens + 3, 1, 2, tokens // 2 + 1]
    pages, table, _ = _setup(lens, 2, dim, 32, bits, seed=tokens)
    q = _q(len(lens), tokens, 2 * group, dim, "fp16", seed=tokens)
    announce(f"attention {tokens} tokens x{group} d={dim} {bits}")
    _run(att, pages, table, lens, q, "whole")
    out = _run(att, pages, table, lens, q, "counts", counts)
    assert bool((out[0] == 0).all()) and bool((out[1, 1:] == 0).all())


@pytest.mark.parametrize("bits,dtype", [(8, "fp16"), (4, "bf16")])
@pytest.mark.parametrize("prefix,tokens,group,batch", [
    (1, 1, 8, 3), (64, 1, 8, 9), (65, 2, 3, 5), (300, 1, 1, 20), (17, 3, 16, 4),
    (130, 1, 4, 40)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prefix(att, bits, dtype, prefix, tokens, group, batch, dim):
    lens = [(7 * b) % 90 for b in range(batch)]
    lens[0] = 0
    pages, table, ptable = _setup(lens, 2, dim, 16, bits, prefix, seed=prefix)
    q = _q(batch, tokens, 2 * group, dim, dtype, seed=prefix)
    announce(f"attention prefix={prefix} tokens={tokens} {batch}x{group} d={dim} {bits}")
    _run(att, pages, table, lens, q, "prefix", prefix=(ptable, prefix))


@pytest.mark.parametrize("lens,tokens,prefix", [
    ([5000, 1, 2311], 1, 0), ([4097], 1, 0), ([777, 3001], 3, 0), ([40, 9], 1, 4500),
    ([1500], 70, 0), ([700, 90], 33, 700)])
@pytest.mark.parametrize("bits", [8, 4])
def test_long(att, lens, tokens, prefix, bits):
    """Axes long enough to be split over workgroups and joined."""
    pages, table, ptable = _setup(lens, 2, 128, 64, bits, prefix, seed=tokens)
    q = _q(len(lens), tokens, 8, 128, "fp16", seed=tokens)
    announce(f"attention long {lens} tokens={tokens} prefix={prefix} {bits}")
    _run(att, pages, table, lens, q, "long", prefix=(ptable, prefix) if prefix else None)


@pytest.mark.parametrize("bits", [8, 4])
def test_missing_pages(att, bits):
    """Table entries that name no page hide their tokens; a length past the
    table sees what the table holds; a row of none of them is empty."""
    pages, table, _ = _setup([200, 200, 90, 64], 2, 64, 16, bits)
    table[0][3] = -1
    table[0][7] = len(pages.k)
    table[1] = [2 ** 31 - 1] * len(table[1])
    table[2] = table[2][:6] + [-1] * (len(table[2]) - 6)
    lens = [200, 200, 90, 5000]
    table[3] = table[3][:4] + [-1] * (len(table[3]) - 4)
    q = _q(4, 2, 6, 64, "fp16")
    announce(f"attention missing pages {bits}")
    out = _run(att, pages, table, lens, q, "missing")
    assert bool((out[1] == 0).all())


@pytest.mark.parametrize("bits", [8, 4])
def test_peaked_and_uneven(att, bits):
    """Scores far apart (one key takes all), value scales over many orders,
    zero scales, the largest fp16 queries, scale of zero and negative."""
    rng = np.random.default_rng(3)
    lens = [150, 150]
    pages, table, _ = _setup(lens, 1, 128, 32, bits, peak=4.0)
    announce(f"attention peaked {bits}")
    _run(att, pages, table, lens, _q(2, 1, 8, 128, "fp16", by=8.0), "peaked")
    for p in table[0]:
        if p >= 0:
            n = min(32, 150 - 32 * table[0].index(p))
            pages.scales[p, :, 1, :n] *= 10.0 ** rng.uniform(-12, 3, (1, n))
    pages.scales[table[0][1], :, 1, 5:9] = 0.0
    pages.scales[table[0][2], :, 0, 5:9] = 0.0
    q = _q(2, 1, 8, 128, "fp16")
    _run(att, pages, table, lens, q, "uneven")
    for s in (0.0, -0.3, 3.0):
        _run(att, pages, table, lens, q, f"scale {s}", scale=s)
    big = torch.full((2, 1, 8, 128), 60000.0).half()
    big[..., ::2] *= -1
    _run(att, pages, table, lens, big, "largest", scale=1e-6)


@pytest.mark.parametrize("dtype", list(DT))
def test_nonfinite(att, dtype):
    """A NaN scale that is seen makes its rows NaN and no others; NaN in one
    query stays in its row; bf16 queries beyond fp16's range."""
    lens = [70, 70, 70]
    pages, table, _ = _setup(lens, 2, 64, 16, 8)
    pages.scales[table[1][2], 0, 0, 3] = np.nan
    pages.scales[table[2][1], 1, 1, 4] = np.nan
    q = _q(3, 2, 4, 64, dtype)
    q[0, 1, 2, 5] = float("nan")
    announce(f"attention nonfinite {dtype}")
    out = _run(att, pages, table, lens, q, "nan")
    assert bool(out[0, 1, 2].isnan().all()) and bool(out[0, 0].isfinite().all())
    if dtype == "bf16":
        big = _q(3, 2, 4, 64, dtype, by=1e30)
        _run(att, pages, table, [20, 20, 16], big, "beyond fp16", scale=1e-31)
        tiny = _q(3, 2, 4, 64, dtype, by=1e-30)
        _run(att, pages, table, [20, 20, 16], tiny, "below fp16", scale=1e29)


def test_strides_streams_graph_and_repeats(att):
    """q as a view of the fused projection, one element off 16 bytes too; out
    given; another stream; a captured graph replayed with new lengths; equal
    bits every time."""
    lens = [1300, 37, 600]
    pages, table, ptable = _setup(lens, 2, 128, 64, 8, 200)
    cache, tab, ln, pt = pages.device(), _ints(table), _ints(lens), _ints(ptable)
    q = _q(3, 1, 16, 128, "fp16").cuda()
    announce("attention strides, streams, graph")
    want = att.forward(q, cache, tab, ln, prefix=(pt, 200))
    for off in (0, 3):
        wide = torch.zeros(3, 1, 3000, dtype=torch.float16, device="cuda")
        view = wide[:, :, off:off + 2048].unflatten(2, (16, 128))
        view.copy_(q)
        assert torch.equal(att.forward(view, cache, tab, ln, prefix=(pt, 200)), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = torch.empty_like(q)
        att.forward_into(q, cache, tab, ln, out, prefix=(pt, 200))
    s.synchronize()
    assert torch.equal(out, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        att.forward_into(q, cache, tab, ln, out, prefix=(pt, 200))
    for now in ([1300, 37, 600], [1, 20, 333], [64, 0, 599], [1300, 37, 600]):
        ln.copy_(_ints(now))
        out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, att.forward(q, cache, tab, ln, prefix=(pt, 200))), now


def test_refusals(att):
    from cudalab_amd.kvcache import KVCache
    c = KVCache.empty(4, 2, 64, 16, 8)
    q = torch.zeros(2, 3, 4, 64, device="cuda").half()
    good = dict(q=q, cache=c, block_table=_ints([[0], [1]]), lengths=_ints([3, 3]))
    for change in (dict(q=q.float()), dict(q=q[..., :32]), dict(q=q[:, :, :3]), dict(q=q[0]),
                   dict(q=q.cpu()), dict(q=q.transpose(2, 3)), dict(cache=c.k), dict(q=None),
                   dict(block_table=_ints([[0]])), dict(lengths=_ints([3])),
                   dict(lengths=_ints([3, 3]).long()), dict(counts=_ints([1])),
                   dict(prefix=(_ints([2]), 17)), dict(prefix=(_ints([2]), -1)),
                   dict(prefix=(_ints([2]).long(), 3)), dict(prefix=(_ints([[2]]), 3)),
                   dict(prefix=(_ints([2]), 2.0)), dict(scale=float("nan")),
                   dict(scale=float("inf"))):
        with pytest.raises(RuntimeError):
            att.forward(**{**good, **change})
    for out in (torch.empty_like(q)[:1], torch.empty_like(q).float(), q,
                torch.empty(2, 3, 4, 128, device="cuda").half()[..., :64]):
        with pytest.raises(RuntimeError):
            att.forward_into(q, c, good["block_table"], good["lengths"], out)
    e = torch.zeros(0, 3, 4, 64, device="cuda").half()
    assert att.forward(e, c, torch.zeros(0, 1, dtype=torch.int32, device="cuda"),
                       _ints([])).shape == e.shape
