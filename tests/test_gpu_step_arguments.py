"""GPU tests of what the calls of a step of many tokens accept and refuse."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import announce

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def att(cuda):
    from cudalab_amd.build import build
    return build("attention")


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def test_a_page_size_that_is_no_whole_number(att):
    """RuntimeError as for any other argument; numpy's whole numbers are ones."""
    args = _ints([[0, 1], [2, 3]]), _ints([0, 0]), _ints([3, 4]), 9
    for page in (16.0, np.float64(16), "16", None):
        with pytest.raises(RuntimeError):
            att.place(*args, page, _ints([5, 6]))
    announce("place, the page size as numpy's")
    assert att.place(*args, np.int64(16), _ints([5, 6])).taken.tolist() == [2]


def test_no_keys_of_any_strides(att):
    """Without keys rows are zeros, whatever the strides of nothing are."""
    q = torch.randn(7, 4, 64, device="cuda").half()
    none = _ints([0, 0])
    wide = torch.zeros(3, 2, 67, device="cuda").half()
    far = torch.zeros(1, dtype=torch.float16, device="cuda").as_strided((0, 2, 64),
                                                                        (2 ** 25, 64, 1))
    for kv in (wide[:0, :, 3:], wide[:0, :, :64], far):
        announce(f"prompt without keys, strides {kv.stride()}")
        got = att.prompt(q, kv, kv, _ints([0, 7]), k_offsets=none)
        assert bool((got == 0).all())


def test_outputs_off_16_bytes(att):
    """An `out` that does not start at 16 bytes is refused, and stays as it was."""
    from cudalab_amd.build import build
    gemm = build("qgemm")
    q = torch.randn(9, 2, 64, device="cuda").half()
    flat = torch.full((9 * 2 * 64 + 8,), 7.0, dtype=torch.float16, device="cuda")
    w = torch.ones(64, 32, dtype=torch.int8, device="cuda")
    x, one = torch.ones(18, 32, dtype=torch.int8, device="cuda"), torch.ones(64, device="cuda")
    for off in (1, 4):
        out = flat[off:off + q.numel()].view(q.shape)
        with pytest.raises(RuntimeError, match="16-byte"):
            att.prompt_into(q, q, q, _ints([0, 9]), out)
        with pytest.raises(RuntimeError, match="16-byte"):
            gemm.forward_into(x, one[:18], w, one, out.view(18, 64))
    torch.cuda.synchronize()
    assert bool((flat == 7).all())
