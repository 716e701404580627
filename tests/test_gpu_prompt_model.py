"""GPU tests of the prompt driver: all operators of a step of many tokens together,
as a model calls them."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from attention_oracle import assert_close, norm_rope, norm_rope_tolerance, quantize
from conftest import announce
from step_oracle import prompt
from test_gpu_decode_context import _pages_of
from test_gpu_tree import tree_attention

pytestmark = pytest.mark.gpu
SIZES = dict(hidden=1024, inter=2048, kv=256)


def _model(batch, room, bits=8, layers=2):
    from cudalab_amd.prompt import PromptModel
    return PromptModel(batch, room, layers, seed=5, cache_bits=bits, **SIZES)


def _x(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).half().cuda()


def _counts(lens):
    return torch.tensor(lens, dtype=torch.int32, device="cuda")


def _qkv(m, x):
    """The first layer's q, k, v of x by the definition: codes, whole sums, FP32."""
    codes, scale = quantize(x.cpu().float().numpy(), 8)
    out = []
    for n in ("q", "k", "v"):
        w, s = (t.cpu() for t in m.weights.layers[0].w[n])
        y = (torch.from_numpy(codes).double() @ w.double().T).float()
        out.append((y * torch.from_numpy(scale)[:, None] * s).half().view(x.size(0), -1, 128))
    return out


@pytest.mark.parametrize("bits", [8, 4])
def test_prompts_against_the_formula(cuda, bits):
    """The first layer's rotated q and k, its cache and o's input; rows behind the
    last sequence leave no trace."""
    lens, spare = [70, 0, 33, 130], 7
    m = _model(4, 150, bits, layers=1)
    x = _x(sum(lens) + spare, 1024)
    seen = {}
    inner = m.att.prompt
    m.att.prompt = lambda q, k, v, o: seen.setdefault("out", inner(
        *(seen.setdefault(n, t) for n, t in (("q", q), ("k", k), ("v", v))), o))
    announce(f"prompts of a layer, {bits} bits")
    try:
        y = m.prompt(x, _counts(lens))
    finally:
        del m.att.prompt
    torch.cuda.synchronize()
    assert y.shape == x.shape and bool(y.isfinite().all())
    assert m.lengths.tolist() == lens
    q, k, v = _qkv(m, x)
    assert torch.equal(seen["v"].cpu(), v)
    positions = torch.tensor([i for n in lens for i in range(n)] + [0] * spare)
    for n, raw, w in (("q", q, m.norms[0][0]), ("k", k, m.norms[0][1])):
        want, mag = norm_rope(raw, w, m.cos, m.sin, positions, 1e-6, False)
        assert_close(seen[n], want.numpy(), norm_rope_tolerance(want, mag, torch.float16).numpy(),
                     n)
    offsets = [0, *np.cumsum(lens).tolist()]
    want, tol = prompt(seen["q"].cpu(), seen["k"].cpu(), seen["v"].cpu(), offsets)
    assert_close(seen["out"], want, tol, "attention")
    host = _pages_of(m.caches[0])
    table = m.table.tolist()
    for which, t in ((0, seen["k"]), (1, seen["v"])):
        codes, scale = quantize(t.cpu().float().numpy(), bits)
        for b, n in enumerate(lens):
            got, there = host.values(table[b], 0, n, which)
            assert there.all()
            at = slice(offsets[b], offsets[b + 1])
            exact = codes[at].astype(np.float64) * scale[at].astype(np.float64)[..., None]
            assert np.array_equal(got, exact.swapaxes(0, 1))


def test_batches_do_not_meet(cuda):
    """A sequence's outputs are the same alone and in a batch."""
    lens = [40, 200, 65]
    x = _x(sum(lens), 1024, seed=1)
    m = _model(3, 210)
    announce("prompts in a batch and alone")
    whole = m.prompt(x, _counts(lens)).clone()
    at = 0
    for n in lens:
        m = _model(1, 210)
        assert torch.equal(m.prompt(x[at:at + n], _counts([n])), whole[at:at + n])
        at += n


@pytest.mark.parametrize("bits", [8, 4])
def test_drafts_are_checked_and_kept(cuda, bits):
    """Trees over the caches against the plain form; what was kept makes the caches
    that the same tokens make one behind another; a second round goes on from there."""
    from cudalab_amd.prompt import chains
    lens, T = [100, 64, 1], 10
    tree, depth = chains(3, T, 2)
    see = np.unpackbits(tree.cpu().numpy().view(np.uint8), axis=-1, bitorder="little")[..., :T]
    m = _model(3, 140, bits)
    m.prompt(_x(sum(lens), 1024, seed=2), _counts(lens))
    x = _x(3, T, 1024, seed=3)
    seen = []
    inner = m.att.forward
    m.att.forward = lambda q, *a, **k: seen.append((q, inner(q, *a, **k))) or seen[-1][1]
    announce(f"drafts checked, {bits} bits")
    try:
        m.check(x, tree, depth)
    finally:
        del m.att.forward
    table = m.table.tolist()
    for i, (q, out) in enumerate(seen):
        want, tol = tree_attention(q.cpu(), _pages_of(m.caches[i]), table, [n + T for n in lens],
                                   see.astype(bool))
        assert_close(out, want, tol, f"layer {i}")
    keep = torch.zeros(3, T, dtype=torch.bool, device="cuda")
    keep[0, 0:8:2] = True          # four tokens of the first chain
    keep[1, 1] = True
    before = [(k.clone(), v.clone()) for k, v in m.drafts]
    m.accept(keep)
    assert m.lengths.tolist() == [104, 65, 1]
    for i, cache in enumerate(m.caches):
        host = _pages_of(cache)
        for which in (0, 1):
            codes, scale = quantize(before[i][which].view(3, T, -1, 128).cpu().float().numpy(),
                                    bits)
            for b in range(3):
                at = keep[b].nonzero()[:, 0].tolist()
                got, there = host.values(table[b], lens[b], len(at), which)
                exact = codes[b, at].astype(np.float64) * scale[b, at].astype(np.float64)[..., None]
                assert there.all() and np.array_equal(got, exact.swapaxes(0, 1))
    y = m.check(x, tree, depth)
    assert bool(y.isfinite().all())


def test_check_in_a_graph(cuda):
    """A captured check replays with new drafts."""
    from cudalab_amd.prompt import chains
    tree, depth = chains(2, 6, 2)
    m = _model(2, 90)
    m.prompt(_x(100, 1024, seed=4), _counts([60, 40]))
    x = _x(2, 6, 1024, seed=5)
    taken = m.taken

    def check():
        m.taken = taken
        return m.check(x, tree, depth)

    check()
    torch.cuda.synchronize()
    announce("a check in a graph")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = check()
    for seed in (6, 7, 8):
        x.copy_(_x(2, 6, 1024, seed=seed))
        g.replay()
        torch.cuda.synchronize()
        got = y.clone()
        assert torch.equal(got, check())


def test_command(cuda, capsys):
    from cudalab_amd import prompt as cmd
    import json
    announce("the prompt command")
    assert cmd.main(["--layers", "1", "--batch", "2", "--tokens", "130", "--drafts", "8",
                     "--steps", "1", "--warmup", "1"]) == 0
    out = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    assert out["prompt_lengths"] == [130, 98] and out["prompt"]["us_per_step"] > 0
    assert out["check"]["drafts"] == 8
