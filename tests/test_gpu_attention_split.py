"""GPU tests of how attention's work is split: many sequences and few, whole
units and broken ones, several groups of rows to a unit, and the two ways that
a call reaches the library."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import announce
from test_gpu_attention import _ints, _q, _run, _setup, att  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("lens", [[(37 * b) % 150 for b in range(150)], [70] * 128,
                                  [0] * 70 + [3] * 3 + [0] * 70 + [600], [0] * 66])
def test_many_sequences(att, bits, lens):                         # noqa: F811
    """More units than lanes that deal them: ragged, equal, mostly empty, empty."""
    pages, table, _ = _setup(lens, 2, 64, 32, bits, seed=len(lens))
    announce(f"attention {len(lens)} sequences, {bits} bits")
    out = _run(att, pages, table, lens, _q(len(lens), 1, 8, 64, "fp16"), "many")
    assert bool((out[[n == 0 for n in lens]] == 0).all())


@pytest.mark.parametrize("bits,dtype", [(8, "fp16"), (4, "bf16")])
@pytest.mark.parametrize("dim,tokens,group,lens", [
    (128, 40, 8, [333, 40]), (64, 70, 7, [500]), (256, 40, 8, [200, 77]),
    (256, 35, 1, [150]), (128, 9, 4, [100] * 66), (64, 33, 1, [90] * 20)])
@pytest.mark.parametrize("uneven", [False, True])
def test_many_rows(att, bits, dtype, dim, tokens, group, lens, uneven):  # noqa: F811
    """Rows enough for whole workgroups, with V scales alike and not."""
    pages, table, _ = _setup(lens, 2, dim, 16, bits, seed=dim + tokens)
    if uneven:
        rng = np.random.default_rng(5)
        by = 10.0 ** rng.uniform(-9, 2, pages.scales[:, :, 1].shape)
        with np.errstate(over="ignore"):                # of stale scales
            pages.scales[:, :, 1] *= by.astype(np.float32)
    announce(f"attention {tokens} tokens x {group} of {len(lens)}, d={dim}, {bits} bits, "
             f"uneven {uneven}")
    _run(att, pages, table, lens, _q(len(lens), tokens, 2 * group, dim, dtype), "rows")


@pytest.mark.parametrize("tokens,lens,prefix", [(1, [2000], 0), (1, [100, 900, 5], 3000),
                                                (50, [60, 1000], 0), (3, [9] * 12, 700)])
def test_checked_path_gives_the_same_bits(att, tokens, lens, prefix):    # noqa: F811
    from cudalab_amd.attention import AttentionExt
    from cudalab_amd.kvcache import KVCache
    assert att._fast is not None
    checked = AttentionExt()
    checked._fast = None
    announce(f"attention both paths, {tokens} tokens, prefix {prefix}")
    pages, table, ptable = _setup(lens, 2, 128, 64, 4, prefix)
    cache, table, n = pages.device(), _ints(table), _ints(lens)
    q = _q(len(lens), tokens, 8, 128, "bf16").cuda()
    ahead = (_ints(ptable), prefix) if prefix else None
    a, b = (x.forward(q, cache, table, n, prefix=ahead, scale=0.1) for x in (att, checked))
    assert torch.equal(a, b)
    k, v = q[:, :, :2], q[:, :, 2:4]
    two = [KVCache.empty(cache.pages, 2, 128, 64, 4) for _ in range(2)]
    got = []
    for x, c in zip((att, checked), two):
        for t in (c.k, c.v, c.scales):
            t.zero_()
        x.append(c, k, v, table, n - tokens)
        got.append((c.k, c.v, c.scales, *x.read(c, table, n - tokens, None, tokens)))
    for s, t in zip(*got):
        assert torch.equal(s, t)
    w = torch.rand(128, device="cuda")
    for s, t in zip(*(x.qk_norm_rope(q[0], q[0, :, :2], w, w) for x in (att, checked))):
        assert torch.equal(s, t)


def test_table_too_long_for_the_deal(att):                        # noqa: F811
    """A table whose keys over all units pass 2^31 steps is refused."""
    from cudalab_amd.kvcache import KVCache
    c = KVCache.empty(1, 64, 64, 256, 4)
    table = torch.zeros(1, 1 << 20, dtype=torch.int32, device="cuda").expand(32, -1)
    q = torch.zeros(32, 1, 64, 64, device="cuda").half()
    announce("attention table too long")
    with pytest.raises(RuntimeError):
        att.forward(q, c, table, _ints([1] * 32))


@pytest.mark.parametrize("bits,dtype", [(8, "bf16"), (4, "fp16")])
@pytest.mark.parametrize("dim,tokens,group,lens", [
    (128, 8, 8, [2500, 60]), (128, 11, 3, [2100]), (64, 5, 13, [2300, 0, 700]),
    (256, 4, 8, [500, 33]), (256, 19, 1, [700])])
def test_few_units_of_several_row_groups(att, bits, dtype, dim, tokens, group, lens):  # noqa: F811
    """Rows of two groups of 16 or 32, over sequences that runs break."""
    pages, table, _ = _setup(lens, 2, dim, 64, bits, seed=dim * tokens)
    announce(f"attention {tokens} tokens x {group}, d={dim}, {bits} bits, few units")
    counts = [tokens, tokens - 2, 1][:len(lens)]
    q = _q(len(lens), tokens, 2 * group, dim, dtype)
    _run(att, pages, table, lens, q, "few units")
    _run(att, pages, table, lens, q, "few units, ragged", counts)
