"""CPU tests of the prompt driver's arguments and helpers."""
from __future__ import annotations

import pytest
import torch

from cudalab_amd import prompt


@pytest.mark.parametrize("args", [["--batch", "0"], ["--tokens", "0"], ["--drafts", "-1"],
                                  ["--layers", "0"], ["--steps", "0"], ["--warmup", "-1"]])
def test_refusals(args, capsys):
    assert prompt.main(args) == 2
    assert "must be" in capsys.readouterr().err


def test_without_a_gpu(capsys):
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible")
    assert prompt.main([]) == 1


def test_chains():
    tree, depth = prompt.chains(2, 70, 3, device="cpu")
    assert tree.shape == (2, 70, 2) and depth[1].tolist() == [t // 3 for t in range(70)]
    for t in (0, 5, 64, 69):
        bits = {64 * w + i for w in range(2) for i in range(64) if tree[1, t, w].item() >> i & 1}
        assert bits == set(range(t % 3, t + 1, 3))


def test_lengths():
    assert prompt.lengths_of(4, 2048) == [2048, 1792, 1536, 1280]
    assert prompt.lengths_of(3, 1) == [1, 1, 1]
