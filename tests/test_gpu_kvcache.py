"""GPU tests of the quantized cache: codes and scales bit for bit against the
definition, nothing else touched, read back exactly."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from attention_oracle import Pages, quantize
from conftest import announce

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def att(cuda):
    from cudalab_amd.build import build
    return build("attention")


def _inputs(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g)
    x *= 10.0 ** torch.randint(-2, 2, (*shape[:3], 1), generator=g)
    return x.to(DT[dtype])


def _append_host(pages, k, v, table, starts, counts):
    B, T = k.shape[:2]
    for which, x in ((0, k), (1, v)):
        codes, scale = quantize(x.float().numpy(), pages.bits)
        for b in range(B):
            for t in range(T if counts is None else min(T, max(0, counts[b]))):
                col, off = divmod(starts[b] + t, pages.page)
                if starts[b] + t < 0 or col >= len(table[b]):
                    continue
                p = table[b][col]
                if 0 <= p < len(pages.k):
                    pages.put(p, off, which, codes[b, t], scale[b, t])


def _same(cache, pages):
    k, v, s = pages.tensors()
    assert torch.equal(cache.k.cpu(), k), "k codes"
    assert torch.equal(cache.v.cpu(), v), "v codes"
    got, want = cache.scales.cpu().numpy(), s.numpy()
    assert (np.isnan(got) == np.isnan(want)).all()
    assert np.array_equal(np.nan_to_num(got, nan=-1.0), np.nan_to_num(want, nan=-1.0)), "scales"


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("d,page,heads", [(64, 16, 3), (128, 64, 2), (256, 32, 1),
                                          (128, 256, 5)])
@pytest.mark.parametrize("tokens", [1, 2, 5, 16, 17, 70])
def test_append_and_read(att, bits, dtype, d, page, heads, tokens):
    starts = [0, 3, page - 1, 2 * page - tokens % 16 - 1]
    cols = (2 * page + tokens) // page + 1
    B = len(starts)
    order = np.random.default_rng(tokens).permutation(B * cols + 1)
    table = [order[b * cols:(b + 1) * cols].tolist() for b in range(B)]
    counts = [tokens, tokens, max(0, tokens - 2), tokens + 9]
    pages = Pages(B * cols + 1, heads, d, page, bits, seed=d + page)
    cache = pages.device()
    k, v = (_inputs((B, tokens, heads, d), dtype, s) for s in (1, 2))
    announce(f"append {bits} bits {dtype} d={d} page={page} heads={heads} tokens={tokens}")
    att.append(cache, k.cuda(), v.cuda(), _ints(table), _ints(starts), _ints(counts))
    _append_host(pages, k, v, table, starts, counts)
    _same(cache, pages)
    gk, gv = att.read(cache, _ints(table), _ints(starts), _ints(counts), tokens + 3, DT[dtype])
    for got, which in ((gk, 0), (gv, 1)):
        for b in range(B):
            n = min(counts[b], tokens + 3)
            want, there = pages.values(table[b], starts[b], n, which)
            want = np.where(there[None, :, None], want, 0.0).astype(np.float32)
            want = torch.from_numpy(want).to(DT[dtype]).transpose(0, 1)
            assert torch.equal(got[b, :n].cpu(), want), (b, which)
            assert bool((got[b, n:] == 0).all())


@pytest.mark.parametrize("bits", [8, 4])
def test_strides_and_alignment(att, bits):
    """k and v as views of a wider projection, and one element off the
    vectors' alignment; tables as columns of a wider one."""
    B, T, H, D, page = 2, 19, 2, 128, 32
    wide = torch.randn(B, T, 6 * H * D + 3, generator=torch.Generator().manual_seed(0)).half()
    table = [[3, 1, 0], [2, 5, 4]]
    for off in (0, 1, 8):
        pages = Pages(6, H, D, page, bits)
        cache = pages.device()
        dev = wide.cuda()

        def view(t, at):
            return t[:, :, at:at + H * D].unflatten(2, (H, D))
        k, v = view(wide, off), view(wide, off + 2 * H * D)
        big = torch.full((2, 9), 77, dtype=torch.int32, device="cuda")
        big[:, :3] = _ints(table)
        announce(f"append views off={off} bits={bits}")
        att.append(cache, view(dev, off), view(dev, off + 2 * H * D), big[:, :3],
                   _ints([5, 40]))
        _append_host(pages, k, v, table, [5, 40], None)
        _same(cache, pages)


@pytest.mark.parametrize("bits", [8, 4])
def test_special_vectors(att, bits):
    """Zeros, tiny, the largest, ties, NaN and Inf: each vector on its own."""
    D, H, T = 64, 1, 12
    x = torch.randn(1, T, H, D, generator=torch.Generator().manual_seed(4))
    x[0, 0] = 0
    x[0, 1] = 2.0 ** -101
    x[0, 2] = 2.0 ** -100
    x[0, 3, 0, 9] = float("nan")
    x[0, 4, 0, 0] = float("inf")
    x[0, 5, 0, 63] = float("-inf")
    x[0, 6] = 3.0e38
    x[0, 7] = torch.arange(D) / 2.0 - 16          # ties, an amax of 16
    x[0, 8, 0, 3] = 3.4e38
    x[0, 9] = -0.0
    pages = Pages(1, H, D, 16, bits)
    cache = pages.device()
    announce(f"append special vectors bits={bits}")
    att.append(cache, x.cuda(), x.flip(1).contiguous().cuda(), _ints([[0]]), _ints([2]))
    _append_host(pages, x, x.flip(1), [[0]], [2], None)
    _same(cache, pages)
    gk, _ = att.read(cache, _ints([[0]]), _ints([2]), None, T, torch.float32)
    assert bool(gk[0, [3, 4, 5]].isnan().all()) and bool((gk[0, [0, 1, 9]] == 0).all())


@pytest.mark.parametrize("bits", [8, 4])
def test_places_out_of_range(att, bits):
    """Positions before the first or past the last page, pages that are none,
    counts of zero and below: nothing written there, zeros read."""
    H, D, page, T = 2, 64, 16, 40
    pages = Pages(4, H, D, page, bits)
    cache = pages.device()
    table = [[0, -1], [4, 1], [2, 2 ** 31 - 1], [-2 ** 31, 3], [3, 0], [1, 2]]
    starts = [0, -5, 10, 0, 2 ** 31 - 20, 0]
    counts = [T, T, T, T, T, -3]
    k, v = _inputs((6, T, H, D), "fp16", 1), _inputs((6, T, H, D), "fp16", 2)
    announce(f"append out of range bits={bits}")
    att.append(cache, k.cuda(), v.cuda(), _ints(table), _ints(starts), _ints(counts))
    _append_host(pages, k, v, table, starts, counts)
    _same(cache, pages)
    gk, gv = att.read(cache, _ints(table), _ints(starts), _ints(counts), T, torch.float32)
    for got, which in ((gk, 0), (gv, 1)):
        for b in range(6):
            n = max(0, counts[b])
            want, there = pages.values(table[b], starts[b], n, which)
            want = np.where(there[None, :, None], want, 0.0).astype(np.float32)
            assert np.array_equal(got[b, :n].cpu().numpy(), want.swapaxes(0, 1)), b
            assert bool((got[b, n:] == 0).all())


def test_empty_calls(att):
    from cudalab_amd.kvcache import KVCache
    c = KVCache.empty(2, 3, 64, 16, 4)
    e = torch.empty(0, 5, 3, 64, device="cuda").half()
    tab = torch.zeros(0, 1, dtype=torch.int32, device="cuda")
    att.append(c, e, e, tab, _ints([]))
    assert att.read(c, tab, _ints([]), None, 5)[0].shape == (0, 5, 3, 64)
    assert att.read(c, _ints([[0]]), _ints([0]), None, 0)[1].shape == (1, 0, 3, 64)


def test_refusals(att):
    from cudalab_amd.kvcache import KVCache
    c = KVCache.empty(4, 2, 64, 16, 8)
    good = dict(cache=c, k=torch.zeros(2, 3, 2, 64, device="cuda").half(),
                v=torch.zeros(2, 3, 2, 64, device="cuda").half(),
                block_table=_ints([[0], [1]]), starts=_ints([0, 0]), counts=_ints([1, 1]))
    k = good["k"]
    for change in (dict(cache=None), dict(k=k.float()), dict(k=k[:1]), dict(k=k.cpu()),
                   dict(k=k.int(), v=k.int()), dict(k=k[..., :32], v=k[..., :32]),
                   dict(k=k.transpose(2, 3), v=k.transpose(2, 3)),
                   dict(k=k[:, :, :1], v=k[:, :, :1]), dict(block_table=_ints([[0]])),
                   dict(block_table=_ints([[0], [1]]).long()), dict(starts=_ints([0])),
                   dict(starts=_ints([0, 0]).long()), dict(counts=_ints([1, 1, 1])),
                   dict(block_table=_ints([0, 1])), dict(starts=torch.zeros(2).int())):
        with pytest.raises(RuntimeError):
            att.append(**{**good, **change})
    for change in (dict(dtype=torch.int8), dict(tokens=-1), dict(tokens=1.5),
                   dict(block_table=_ints([[0]])), dict(cache=c.k), dict(tokens=2 ** 31)):
        with pytest.raises(RuntimeError):
            att.read(**{**dict(cache=c, block_table=good["block_table"], counts=None,
                               starts=good["starts"], tokens=3), **change})
    for bad in ((c.k, c.k, c.scales), (c.k, c.v, c.scales[:, :, :1]), (c.k.cpu(), c.v, c.scales),
                (c.k.view(torch.uint8), c.v, c.scales), (c.k, c.v, c.scales.half()),
                (c.k[..., :32], c.v, c.scales), (c.k[:2], c.v, c.scales),
                (c.k.transpose(0, 1), c.v, c.scales)):
        with pytest.raises(RuntimeError):
            KVCache(*bad)
    for bad in ((4, 2, 80), (4, 2, 64, 48), (4, 2, 64, 16, 5), (0, 2, 64), (2, 0, 64)):
        with pytest.raises(RuntimeError):
            KVCache.empty(*bad)
