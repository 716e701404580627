"""GPU tests of the attention of packed sequences against the plain form in 64
bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from attention_oracle import assert_close
from conftest import announce
from step_oracle import prompt

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def att(cuda):
    from cudalab_amd.build import build
    return build("attention")


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _offsets(lens):
    return [0, *np.cumsum(lens).tolist()]


def _inputs(rows, keys, hq, h, d, dtype, seed=0, by=1.5):
    g = torch.Generator().manual_seed(seed)
    return tuple((torch.randn(n, heads, d, generator=g) * s).to(DT[dtype])
                 for n, heads, s in ((rows, hq, by), (keys, h, 1.0), (keys, h, 1.0)))


def _check(att, q, k, v, offsets, k_offsets=None, causal=True, scale=None, what=""):
    announce(f"prompt {what} {q.dtype} q {tuple(q.shape)} k {tuple(k.shape)} causal={causal} "
             f"offsets {offsets[:9]} {k_offsets and k_offsets[:9]}")
    got = att.prompt(q.cuda(), k.cuda(), v.cuda(), _ints(offsets),
                     k_offsets=None if k_offsets is None else _ints(k_offsets), causal=causal,
                     scale=scale)
    want, tol = prompt(q, k, v, offsets, k_offsets, causal, scale)
    assert_close(got, want, tol, what)
    return got


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lens,hq,h", [
    ([1], 1, 1), ([2, 0, 1, 33], 4, 2), ([63, 64, 65], 3, 3), ([31, 32, 127, 128, 129], 8, 1),
    ([300], 2, 1), ([0, 0, 5, 0], 7, 1), ([257, 1, 1, 200], 8, 8), ([7] * 70, 2, 2)])
def test_lengths_and_heads(att, dtype, d, lens, hq, h):
    rows = sum(lens)
    q, k, v = _inputs(rows, rows, hq, h, d, dtype)
    _check(att, q, k, v, _offsets(lens))
    _check(att, q, k, v, _offsets(lens), causal=False)


@pytest.mark.parametrize("dtype,d", [("fp16", 128), ("bf16", 64), ("bf16", 256)])
@pytest.mark.parametrize("hq,h", [(8, 2), (4, 1), (6, 3), (14, 7), (16, 2), (12, 3)])
@pytest.mark.parametrize("lens", [[20] * 9 + [0, 1, 33], [50, 64, 3, 0, 65, 129], [1] * 40,
                                  [300] + [5] * 30])
def test_short_sequences_of_grouped_heads(att, dtype, d, hq, h, lens):
    """Heads of a group share a workgroup where sequences are short, also with a
    long one among them, keys ahead, rows of no sequence, and NaN that few rows see."""
    rows = sum(lens)
    q, k, v = _inputs(rows + 3, rows + 3, hq, h, d, dtype, 14)
    offsets = _offsets(lens)
    _check(att, q, k, v, offsets)
    seen = [n + 7 * (i % 3) for i, n in enumerate(lens)]
    q, k, v = _inputs(rows, sum(seen), hq, h, d, dtype, 15)
    _check(att, q, k, v, offsets, _offsets(seen))
    clean = att.prompt(q[:rows].cuda(), k[:rows].cuda(), v[:rows].cuda(), _ints(offsets)).cpu()
    bad = offsets[1] - 1
    v[bad, 0] = float("nan")
    got = att.prompt(q[:rows].cuda(), k[:rows].cuda(), v[:rows].cuda(), _ints(offsets)).cpu()
    assert bool(got[bad, :hq // h].isnan().all())
    got[bad, :hq // h] = clean[bad, :hq // h]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("dtype,d", [("fp16", 128), ("bf16", 64), ("bf16", 256)])
def test_more_and_fewer_keys_than_queries(att, dtype, d):
    """Chunks with keys of earlier ones ahead; fewer keys than queries leave
    rows that see nothing."""
    lens = [5, 70, 0, 130, 1, 40, 200]
    seen = [105, 70, 9, 129, 513, 0, 64]
    q, k, v = _inputs(sum(lens), sum(seen), 6, 2, d, dtype, 1)
    for causal in (True, False):
        _check(att, q, k, v, _offsets(lens), _offsets(seen), causal)


@pytest.mark.parametrize("dtype,d", [("fp16", 128), ("bf16", 64), ("bf16", 256)])
def test_waves_with_fewer_keys_than_others(att, dtype, d):
    """Waves that have no rows, or whose rows see none of a tile's keys, load their
    part of the next tile all the same, and the others wait for it."""
    lens = [1, 5, 33, 65, 97, 33, 64, 128] * 12
    keys = [194, 65, 130, 131, 300, 34, 129, 161] * 12
    for seed in range(3):
        q, k, v = _inputs(sum(lens), sum(keys), 8, 4, d, dtype, 40 + seed)
        _check(att, q, k, v, _offsets(lens), _offsets(keys), what=f"seed {seed}")


@pytest.mark.parametrize("dtype,d", [("fp16", 128), ("bf16", 128), ("fp16", 64), ("bf16", 256)])
def test_many_rows(att, dtype, d):
    """Enough rows for the larger workgroups, of lengths that end anywhere."""
    lens = [1111, 1025, 512, 3, 700, 1300]
    q, k, v = _inputs(sum(lens), sum(lens), 32, 2, d, dtype, 2)
    q, k, v = q[:, :8].contiguous(), k[:, :2].contiguous(), v[:, :2].contiguous()
    _check(att, q, k, v, _offsets(lens))
    wide = torch.cat([q, q.flip(1), q, q * 2, q, -q], 1)
    got = att.prompt(wide.cuda(), k.cuda(), v.cuda(), _ints(_offsets(lens)))
    # every head over the keys of its group: the first 24 of head 0
    want, tol = prompt(wide[:, 8:12], k[:, :1], v[:, :1], _offsets(lens))
    assert_close(got[:, 8:12], want, tol, "many heads")


def test_views_alignment_and_strides(att):
    """q, k and v side by side in one tensor; one element off 16 bytes; heads
    and tokens swapped; a single token with any stride."""
    rows, hq, h, d = 150, 4, 2, 128
    for off in (0, 8, 1):
        wide = torch.randn(rows, (hq + 2 * h) * d + 16,
                           generator=torch.Generator().manual_seed(3)).half().cuda()
        q = wide[:, off:off + hq * d].view(rows, hq, d)
        k = wide[:, off + hq * d:off + (hq + h) * d].view(rows, h, d)
        v = wide[:, off + (hq + h) * d:off + (hq + 2 * h) * d].view(rows, h, d)
        want, tol = prompt(q.cpu(), k.cpu(), v.cpu(), [0, 70, 150])
        announce(f"prompt views off={off}")
        assert_close(att.prompt(q, k, v, _ints([0, 70, 150])), want, tol, f"off {off}")
    q, k, v = _inputs(90, 90, 4, 2, 64, "bf16", 4)
    swapped = [x.transpose(0, 1).contiguous().cuda().transpose(0, 1) for x in (q, k, v)]
    want, tol = prompt(q, k, v, [0, 90])
    assert_close(att.prompt(*swapped, _ints([0, 90])), want, tol, "swapped")
    one = [x.cuda()[:1].as_strided((1, x.shape[1], 64), (3, 64, 1)) for x in (q, k, v)]
    want, tol = prompt(q[:1], k[:1], v[:1], [0, 1])
    assert_close(att.prompt(*one, _ints([0, 1])), want, tol, "one token")
    # keys far apart
    want, tol = prompt(q[:3, :1], k[:3, :1], v[:3, :1], [0, 3])
    for n in (2 ** 24, 2 ** 24 + 64):
        far = torch.zeros(3, n, dtype=torch.bfloat16, device="cuda")
        far[:, :64], far[:, 64:128] = k[:3, 0].cuda(), v[:3, 0].cuda()
        announce(f"prompt token stride {n}")
        assert_close(att.prompt(q[:3, :1].cuda(), far[:, None, :64], far[:, None, 64:128],
                                _ints([0, 3])), want, tol, f"token stride {n}")


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 1e-6, 3.0])
def test_scales(att, scale):
    q, k, v = _inputs(140, 140, 2, 1, 64, "fp16", 5)
    _check(att, q, k, v, [0, 100, 140], scale=scale, what=f"scale {scale}")


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("d", [64, 128, 256])
def test_what_is_not_seen_leaves_no_trace(att, dtype, d):
    """NaN and Inf in keys and values: rows ahead of them, and other sequences,
    are as without; rows that see them are as the formula says."""
    lens = [130, 200, 40]
    offsets = _offsets(lens)
    q, k, v = _inputs(sum(lens), sum(lens), 2, 1, d, dtype, 6)
    clean, _ = prompt(q, k, v, offsets)
    for what, value, places in (("v", float("nan"), (100, 130 + 64)), ("v", float("inf"), (129,)),
                                ("k", float("nan"), (65, 131)), ("v", float("-inf"), (369,)),
                                ("k", float("inf"), (64,))):
        kk, vv = k.clone(), v.clone()
        for p in places:
            (kk if what == "k" else vv)[p, 0, 3 if what == "k" else slice(1, d, 7)] = value
        announce(f"prompt {value} in {what} {dtype} {d}")
        got = att.prompt(q.cuda(), kk.cuda(), vv.cuda(), _ints(offsets)).double().cpu().numpy()
        want, tol = prompt(q, kk, vv, offsets)
        spoilt = np.zeros(sum(lens), bool)
        for p in places:
            b = np.searchsorted(offsets, p, side="right") - 1
            spoilt[p:offsets[b + 1]] = True
        err = np.abs(got - clean)
        assert (err[~spoilt] <= tol[~spoilt]).all(), (what, value)
        # seen: not finite in the dims that the value is in, the others as they are
        if what == "v":
            bad = ~np.isfinite(got[spoilt])
            assert bad[..., 1::7].all()
            rest = np.ones(d, bool)
            rest[1::7] = False
            assert (err[spoilt][..., rest] <= tol[spoilt][..., rest]).all()
        elif np.isnan(value):
            assert np.isnan(got[spoilt]).all()


@pytest.mark.parametrize("dtype", list(DT))
def test_queries_apart(att, dtype):
    """Rows of very different size, and one with NaN and Inf, side by side: each
    is its own."""
    q, k, v = _inputs(96, 96, 2, 2, 128, dtype, 7)
    q *= 2.0 ** torch.randint(-12, 4, (96, 1, 1), generator=torch.Generator().manual_seed(1))
    q[40, 0, 5], q[50, 1, 0] = float("nan"), float("inf")
    announce(f"prompt rows apart {dtype}")
    got = att.prompt(q.cuda(), k.cuda(), v.cuda(), _ints([0, 96])).cpu()
    with np.errstate(all="ignore"):
        want, tol = prompt(q, k, v, [0, 96])
    assert bool(got[40, 0].isnan().all()) and not bool(got[50, 1].isfinite().all())
    keep = torch.ones(96, 2, dtype=torch.bool)
    keep[40, 0] = keep[50, 1] = False
    assert_close(got[keep], want[keep.numpy()], tol[keep.numpy()], "others")


def test_rows_of_no_sequence(att):
    """Rows ahead of the first offset and behind the last are zeros; offsets past
    the tensor are cut."""
    q, k, v = _inputs(700, 700, 4, 2, 64, "fp16", 8)
    q[600:], k[600:], v[600:] = float("nan"), float("nan"), float("nan")
    for offsets in ([0, 100, 250], [130, 200, 330, 330, 599], [0, 0], [600, 600]):
        got = _check(att, q, k, v, offsets, what="rows of no sequence")
        assert bool((got[offsets[-1]:] == 0).all()) and bool((got[:offsets[0]] == 0).all())
    want, tol = prompt(q[:500], k[:500], v[:500], [0, 300, 500])
    announce("prompt offsets past the tensor")
    got = att.prompt(q[:500].cuda(), k[:500].cuda(), v[:500].cuda(),
                     _ints([-7, 300, 2 ** 31 - 1]))
    assert_close(got, want, tol, "cut")
    out = torch.full((500, 4, 64), 7.0, dtype=torch.float16, device="cuda")
    att.prompt_into(q[:500].cuda(), k[:500].cuda(), v[:500].cuda(), _ints([0, 300, 500]), out)
    assert torch.equal(out, got)


def test_many_sequences(att):
    """More sequences than lanes: 1, 2 and 0 tokens, and a few long ones."""
    lens = [(i * 7) % 3 for i in range(400)]
    lens[70], lens[300], lens[399] = 300, 140, 65
    q, k, v = _inputs(sum(lens), sum(lens), 2, 1, 64, "bf16", 9)
    _check(att, q, k, v, _offsets(lens), what="many")


@pytest.mark.parametrize("batch", [60, 61, 62, 63, 64, 257, 1500])
def test_batches_around_a_wave(att, batch):
    """Lengths around whole tiles and empty ones, rows ahead of the first and behind
    the last sequence."""
    rng = np.random.default_rng(batch)
    lens = rng.choice([0, 0, 1, 2, 5, 31], batch)
    lens[rng.permutation(batch)[:8]] = [127, 128, 129, 255, 256, 257, 300, 1]
    offsets = [9, *(9 + np.cumsum(lens)).tolist()]
    q, k, v = _inputs(offsets[-1] + 150, offsets[-1] + 150, 2, 1, 64, "fp16", 12)
    got = _check(att, q, k, v, offsets, what=f"{batch} sequences")
    assert bool((got[:9] == 0).all()) and bool((got[offsets[-1]:] == 0).all())


def test_graph_replays_with_new_offsets(att):
    q, k, v = (x.cuda() for x in _inputs(600, 600, 4, 2, 128, "fp16", 10))
    offsets = _ints([0, 10, 600])
    out = torch.empty_like(q)
    att.prompt_into(q, k, v, offsets, out)
    torch.cuda.synchronize()
    announce("prompt in a graph")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        att.prompt_into(q, k, v, offsets, out)
    for new in ([0, 300, 600], [0, 64, 65], [0, 599, 599], [0, 1, 600]):
        offsets.copy_(_ints(new))
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, att.prompt(q, k, v, _ints(new)))
        want, tol = prompt(q.cpu(), k.cpu(), v.cpu(), new)
        assert_close(got, want, tol, f"replay {new}")


def test_streams_and_repeats(att):
    q, k, v = (x.cuda() for x in _inputs(300, 300, 8, 2, 64, "bf16", 11))
    offsets = _ints([0, 200, 300])
    a = att.prompt(q, k, v, offsets)
    torch.cuda.synchronize()
    announce("prompt on two streams")
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in sides:
        with torch.cuda.stream(s):
            got.append(att.prompt(q, k, v, offsets))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for b in got)


def test_empty_and_refusals(att):
    q, k, v = (x.cuda() for x in _inputs(6, 6, 4, 2, 64, "fp16"))
    o = _ints([0, 6])
    assert att.prompt(q[:0], k[:0], v[:0], _ints([0, 0])).shape == (0, 4, 64)
    assert bool((att.prompt(q, k, v, _ints([0])) == 0).all())
    assert bool((att.prompt(q, k[:0], v[:0], o, k_offsets=_ints([0, 0])) == 0).all())
    good = dict(q=q, k=k, v=v, offsets=o)
    for change in (dict(q=None), dict(q=q.float(), k=k.float(), v=v.float()), dict(k=k.bfloat16()),
                   dict(q=q.cpu()), dict(k=k[:5]), dict(v=v[:5]), dict(q=q[:, :3]),
                   dict(q=q[..., :32], k=k[..., :32], v=v[..., :32]), dict(q=q[None]),
                   dict(q=q.transpose(1, 2)), dict(k=k[:, :0], v=v[:, :0]),
                   dict(offsets=o.long()), dict(offsets=o[:0]), dict(offsets=o[None]),
                   dict(offsets=[0, 6]), dict(offsets=_ints([0, 3, 6, 6])[::2]),
                   dict(k_offsets=_ints([0, 3, 6])), dict(k_offsets=o.cpu()), dict(scale="x"),
                   dict(scale=float("nan")), dict(scale=float("inf"))):
        with pytest.raises(RuntimeError):
            att.prompt(**{**good, **change})
    for out in (None, torch.empty_like(q)[:5], torch.empty_like(q).float(), q.transpose(0, 1),
                torch.empty_like(q).cpu(), q):
        with pytest.raises(RuntimeError):
            att.prompt_into(**good, out=out)
