"""GPU tests of attention where keys without a value, or with a very small
one, stand beside keys with a large one: they stay in the denominator."""
from __future__ import annotations

import numpy as np
import pytest

from attention_oracle import Pages
from conftest import announce
from test_gpu_attention import _q, _run, att  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

LOG2E = 1.4426950408889634


def _pages(n, at, bits, dim, big, below, other, seed=0):
    """One sequence of n tokens of one head and a q of ones of which key `at`
    has V scale `big` and the others `other`, scores `below` bits lower."""
    rng = np.random.default_rng(seed)
    page = 64
    pages = Pages(-(-n // page), 1, dim, page, bits, seed)
    pages.k[:] = 1
    pages.scales[:, :, 0] = 30.0 - below
    pages.scales[:, :, 1] = other
    if other == 0:
        pages.v[:] = 0
    p, off = divmod(at, page)
    pages.scales[p, 0, 0, off], pages.scales[p, 0, 1, off] = 30.0, big
    top = 127 if bits == 8 else 7
    pages.v[p, 0, off] = rng.integers(1, top + 1, dim)
    return pages, [list(range(len(pages.k)))]


def _check(att, n, at, bits, dim, tokens, group, big, below, other, dtype):  # noqa: F811
    pages, table = _pages(n, at, bits, dim, big, below, other)
    q = _q(1, tokens, group, dim, dtype)
    q[:] = 1.0                               # scores in bits: K's scale
    _run(att, pages, table, [n], q, f"{n} keys, {at} of {big}, {below} below of {other}",
         scale=1.0 / dim / LOG2E)


@pytest.mark.parametrize("tokens,group", [(1, 4), (40, 4)])
@pytest.mark.parametrize("bits,dtype,big,below,n", [
    (4, "fp16", 8571.0, 13.0, 4000), (8, "fp16", 500.0, 13.0, 4000),
    (8, "bf16", 16.0, 15.0, 9000), (8, "bf16", 2.0 ** 27, 6.0, 700),
    (4, "bf16", 1e20, 4.0, 300), (8, "bf16", 1e26, 3.0, 300), (8, "bf16", 1e30, 1.0, 100)])
@pytest.mark.parametrize("where", ["first", "middle", "last"])
def test_keys_without_a_value(att, tokens, group, bits, dtype, big, below, n, where):  # noqa: F811
    """Thousands of keys of scale zero some bits below one of a large scale."""
    last = n - tokens                        # what every row sees
    at = dict(first=0, middle=last // 2 + 5, last=last)[where]
    announce(f"attention {n} keys without a value, {big} at {at}, {tokens} tokens, {bits}")
    _check(att, n, at, bits, 128, tokens, group, big, below, 0.0, dtype)


@pytest.mark.parametrize("dim,tokens,group", [(64, 1, 16), (256, 1, 4), (64, 33, 2),
                                              (256, 40, 4)])
@pytest.mark.parametrize("big,below,other", [(2.0 ** 20, 9.0, 0.0), (2.0 ** 20, 9.0, 1e-8),
                                             (1e15, 5.0, 1e-15), (1.0, 5.0, 1e-24),
                                             (1e-20, 5.0, 0.0), (1e-24, 7.0, 1e-24)])
def test_scales_far_apart(att, dim, tokens, group, big, below, other):       # noqa: F811
    """Other heads and scales: tiny ones beside large ones, all tiny."""
    announce(f"attention scales {big} and {other}, d={dim} {tokens}x{group}")
    for at in (0, 700):
        _check(att, 1500, at, 8, dim, tokens, group, big, below, other, "bf16")
