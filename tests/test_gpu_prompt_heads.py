"""GPU tests of which workgroup takes which heads: every head of calls whose
workgroups are dealt to the XCDs by heads, over outputs that held NaN."""
from __future__ import annotations

import pytest
import torch

from attention_oracle import assert_close
from conftest import announce
from step_oracle import prompt
from test_gpu_prompt import DT, _inputs, _ints, _offsets

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def att(cuda):
    from cudalab_amd.build import build
    return build("attention")


# runs of heads: 48, 32, 64, 16 (pairs of 32) and 16 (fours of 64), 40, 12 (not dealt)
@pytest.mark.parametrize("hq,h,lens", [
    (48, 2, [130, 257, 70]), (32, 4, [300, 129]), (64, 8, [200, 150]), (32, 32, [140, 90]),
    (32, 4, [60, 50, 64, 1, 33]), (64, 16, [20] * 9 + [31]), (40, 8, [129, 140]),
    (12, 4, [128, 131])])
@pytest.mark.parametrize("dtype,d", [("fp16", 64), ("bf16", 128), ("fp16", 256)])
def test_every_head(att, dtype, d, hq, h, lens):
    rows = sum(lens)
    q, k, v = _inputs(rows, rows, hq, h, d, dtype, 50)
    offsets = _offsets(lens)
    out = torch.full(q.shape, float("nan"), dtype=DT[dtype], device="cuda")
    announce(f"prompt of {hq}/{h} heads of {d}, {dtype}, {lens}")
    att.prompt_into(q.cuda(), k.cuda(), v.cuda(), _ints(offsets), out)
    want, tol = prompt(q, k, v, offsets)
    assert_close(out, want, tol, "every head")
