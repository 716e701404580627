"""GPU tests of attention's deal of many rows: the join of eight rows at a
time, and tables whose keys are too many."""
from __future__ import annotations

import pytest
import torch

from attention_oracle import assert_close, attention
from conftest import announce
from test_gpu_attention import _ints, _q, _setup, att  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits,dtype", [(8, "fp16"), (4, "bf16")])
@pytest.mark.parametrize("tokens,group,dim,lens", [
    # rows of no multiple of eight; sequences of nothing, of one key, shorter
    # than the new tokens, and long enough for several runs
    (911, 3, 64, [1500, 0, 950, 3000, 1, 911]),
    (1031, 4, 128, [2600, 1100, 7, 0]),
    (1025, 4, 256, [1300, 0, 600, 1025])])
def test_join_of_eight_rows(att, bits, dtype, tokens, group, dim, lens):  # noqa: F811
    heads = 2
    assert tokens * group * heads * len(lens) >= 8 * 4 * 4 * 256     # rows enough for eight
    pages, table, _ = _setup(lens, heads, dim, 64, bits, seed=tokens)
    q = _q(len(lens), tokens, heads * group, dim, dtype, seed=dim)
    counts = [tokens, 500, tokens - 9, tokens, 3, tokens][:len(lens)]
    for what, n in (("whole", None), ("counts", counts)):
        announce(f"attention {tokens} tokens x {group} of {len(lens)}, d={dim} {bits}, {what}")
        out = att.forward(q.cuda(), pages.device(), _ints(table), _ints(lens),
                          None if n is None else _ints(n)).cpu()
        assert bool(out.isfinite().all())
        for b, length in enumerate(lens):
            own = tokens if n is None else n[b]
            # rows t see up to length - own + t; the first that see anything too
            first = max(0, own - length)
            some = {0, 1, first - 1, first, first + 1, own // 2, own - 8, own - 2, own - 1}
            for t in sorted(t for t in some if 0 <= t < own):
                want, tol = attention(q[b:b + 1, t:t + 1], pages, table[b:b + 1],
                                      [length - own + t + 1])
                assert_close(out[b:b + 1, t:t + 1], want, tol, f"{what} {b} {t}")
            assert bool((out[b, :min(first, own)] == 0).all())
            assert bool((out[b, own:] == 0).all())


def test_table_of_too_many_keys(att):                                # noqa: F811
    """Keys over all units past 2^31 steps, in a table of valid strides."""
    from cudalab_amd.kvcache import KVCache
    c = KVCache.empty(1, 64, 64, 256, 4)
    table = torch.zeros(32, 1 << 20, dtype=torch.int32, device="cuda")
    q = torch.zeros(32, 1, 64, 64, device="cuda").half()
    announce("attention of too many keys")
    with pytest.raises(RuntimeError, match="too many for one call"):
        att.forward(q, c, table, _ints([1] * 32))
