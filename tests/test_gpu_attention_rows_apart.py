"""GPU tests of attention where rows that are worked on together have queries
of very different size: each row's result is its own."""
from __future__ import annotations

import pytest
import torch

from conftest import announce
from test_gpu_attention import _q, _run, _setup, att  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("tokens,group,dim", [(4, 4, 128), (3, 8, 64), (5, 3, 256), (40, 4, 128),
                                              (33, 4, 64), (40, 4, 256), (9, 3, 128)])
@pytest.mark.parametrize("junk", [1e12, -3e38, float("nan"), float("inf")])
def test_rows_past_the_count(att, bits, tokens, group, dim, junk):   # noqa: F811
    """What a padded q holds past the counts reaches no result."""
    lens, counts = [200, 70, 131, 90], [1, 2, tokens, 0]
    pages, table, _ = _setup(lens, 2, dim, 32, bits, seed=dim + tokens)
    q = _q(4, tokens, 2 * group, dim, "bf16", seed=tokens)
    for b, n in enumerate(counts):
        q[b, n:] = junk
        q[b, n:, ::2, 1::3] *= 0.125
    announce(f"attention past the count {junk}, {tokens}x{group} d={dim} {bits}")
    out = _run(att, pages, table, lens, q, f"junk {junk}", counts)
    for b, n in enumerate(counts):
        assert bool((out[b, n:] == 0).all())


@pytest.mark.parametrize("bits,dim", [(8, 128), (4, 64), (8, 256)])
@pytest.mark.parametrize("batch,group", [(5, 3), (40, 4)])
@pytest.mark.parametrize("apart", [2.0 ** 40, 1e12, 2.0 ** -40])
def test_sequences_apart_over_a_prefix(att, bits, dim, batch, group, apart):  # noqa: F811
    """One sequence's queries many times the others', over keys of all."""
    lens = [(7 * b) % 50 for b in range(batch)]
    pages, table, ptable = _setup(lens, 2, dim, 16, bits, 150, seed=batch)
    q = _q(batch, 1, 2 * group, dim, "bf16", seed=batch)
    q[batch // 2] *= apart
    announce(f"attention prefix, a sequence {apart} times the others, {batch}x{group} d={dim}")
    for scale in (None, dim ** -0.5 / max(apart, 1.0)):
        _run(att, pages, table, lens, q, f"apart, scale {scale}", prefix=(ptable, 150),
             scale=scale)


@pytest.mark.parametrize("bits,dtype,by", [(8, "bf16", 1e9), (4, "bf16", 1e25), (8, "fp16", 2e4)])
@pytest.mark.parametrize("tokens,group,dim", [(1, 16, 128), (2, 16, 64), (1, 8, 256),
                                              (70, 2, 128), (40, 4, 256)])
def test_heads_apart(att, bits, dtype, by, tokens, group, dim):      # noqa: F811
    """Heads of one sequence by turns large, ordinary and small."""
    lens = [300, 90]
    pages, table, _ = _setup(lens, 2, dim, 64, bits, seed=group)
    q = _q(2, tokens, 2 * group, dim, dtype, seed=group)
    q[:, :, 0::3] *= by
    q[:, :, 1::3] /= by
    announce(f"attention heads {by} apart, {dtype} {tokens}x{group} d={dim} {bits}")
    for scale in (None, dim ** -0.5 / by):
        _run(att, pages, table, lens, q, f"heads apart, scale {scale}", scale=scale)


def test_largest_queries(att):                                       # noqa: F811
    """bf16's largest and smallest numbers, scores in range by the scale."""
    lens = [100, 33]
    for tokens in (1, 40):
        pages, table, _ = _setup(lens, 1, 128, 32, 8, seed=1)
        q = _q(2, tokens, 6, 128, "bf16")
        q[:, :, 0] = q[:, :, 0].sign() * 3.3e38
        q[:, :, 1] = 1e-38
        announce(f"attention largest queries, {tokens} tokens")
        _run(att, pages, table, lens, q, "largest", scale=2.0 ** -129)
