"""GPU tests of trees of many rows: the join of a wave to a row, units of 128 rows
of calls that would have 256, all head sizes, a prefix."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_tree import _ancestors, _case, _check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def att(cuda):
    from cudalab_amd.build import build
    return build("attention")


# rows of a key head: 336 (three units of 128), 272 (three), 512 (two of 256), 224
# (two of 128 of heads of 256, one of 256 else); all of them 4096 and more over the call
@pytest.mark.parametrize("B,T,hq,h,lengths", [
    (4, 42, 32, 4, [42, 700, 300, 90]), (4, 34, 32, 4, [600, 34, 35, 64]),
    (4, 64, 16, 2, [64, 500, 129, 70]), (5, 28, 32, 4, [28, 400, 130, 1, 64])])
@pytest.mark.parametrize("bits,d,page,dtype", [(8, 128, 64, "fp16"), (4, 64, 32, "bf16"),
                                               (8, 256, 16, "bf16"), (4, 128, 128, "fp16")])
def test_many_rows(att, B, T, hq, h, lengths, bits, d, page, dtype):
    rng, pages, table, q, spare = _case(B, T, hq, h, d, page, bits, dtype, lengths, 11)
    see = _ancestors(B, T, rng)
    assert B * T * hq >= 4096
    _check(att, q, pages, table, lengths, see, what="many rows")
    counts = [T, T // 2, T, 0, T][:B]
    _check(att, q, pages, table, lengths, see, counts, (spare, page + 5), what="and a prefix")


def test_rows_that_see_nothing(att):
    """Among many rows: no bits at all, and sequences without tokens."""
    B, T = 4, 33
    rng, pages, table, q, _ = _case(B, T, 32, 4, 64, 32, 8, "fp16", [33, 200, 0, 70], 12)
    see = rng.random((B, T, T)) < 0.4
    see[:, 5] = False
    got = _check(att, q, pages, table, [33, 200, 0, 70], see, what="nothing seen").cpu().numpy()
    assert np.array_equal(got[0, 5], np.zeros_like(got[0, 5])) and not got[2].any()
