"""GPU tests of the per-head norms with the rotation against the formula in
64 bits: types, head sizes on and off the vector kernel, strides, in place,
positions out of the tables."""
from __future__ import annotations

import pytest
import torch

from attention_oracle import UNIT, assert_close, norm_rope, norm_rope_tolerance
from conftest import announce

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def att(cuda):
    from cudalab_amd.build import build
    return build("attention")


def _tables(rows, rot, seed=0):
    g = torch.Generator().manual_seed(seed)
    ang = torch.rand(rows, rot // 2, generator=g) * 100 - 50
    return ang.cos(), ang.sin()


def _check(got, x, w, cos, sin, pos, inter, what, eps=1e-6):
    y, mag = norm_rope(x, w, cos, sin, pos, eps, inter)
    assert_close(got, y.numpy(), norm_rope_tolerance(y, mag, x.dtype).numpy(), what)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("tokens,hq,hkv,d,rot", [
    (1, 64, 8, 128, 128), (3, 5, 1, 128, 128), (2, 1, 1, 64, 64), (5, 3, 2, 64, 32),
    (4, 7, 3, 256, 256), (3, 2, 2, 80, 80), (2, 4, 1, 96, 48), (2, 3, 1, 512, 512),
    (2, 2, 1, 1024, 1024), (3, 2, 1, 2, 2), (5, 3, 1, 70, 6), (2, 3, 3, 72, 24),
    (2, 2, 1, 576, 64), (301, 9, 3, 128, 64), (2000, 40, 8, 64, 64)])
def test_norm_rope(att, dtype, inter, tokens, hq, hkv, d, rot):
    announce(f"norm_rope {dtype} inter={inter} {tokens}x({hq}+{hkv})x{d} rot={rot}")
    g = torch.Generator().manual_seed(tokens + d)
    dt = DT[dtype]
    q = torch.randn(tokens, hq, d, generator=g).to(dt)
    k = (torch.randn(tokens, hkv, d, generator=g) * 30).to(dt)
    qw, kw = ((1 + 0.3 * torch.randn(d, generator=g)).to(dt) for _ in range(2))
    cos, sin = _tables(50, rot)
    pos = torch.randint(0, 50, (tokens,), generator=g, dtype=torch.int32)
    dev = [t.cuda() for t in (q, k, qw, kw, cos, sin, pos)]
    gq, gk = att.qk_norm_rope(*dev, interleaved=inter)
    assert gq.is_contiguous() and gq.dtype == dt and gk.shape == k.shape
    _check(gq, q, qw, cos, sin, pos, inter, "q")
    _check(gk, k, kw, cos, sin, pos, inter, "k")


@pytest.mark.parametrize("weights,tables", [("both", False), ("none", True), ("q", True),
                                            ("k", False), ("f32", True)])
def test_parts_left_out(att, weights, tables):
    g = torch.Generator().manual_seed(3)
    q, k = torch.randn(6, 4, 128, generator=g).half(), torch.randn(6, 2, 128, generator=g).half()
    wt = torch.float32 if weights == "f32" else torch.float16
    qw = torch.randn(128, generator=g).to(wt) if weights in ("both", "q", "f32") else None
    kw = torch.randn(128, generator=g).to(wt) if weights in ("both", "k", "f32") else None
    cos, sin = _tables(9, 128) if tables else (None, None)
    pos = torch.tensor([0, 8, 3, 3, 1, 7], dtype=torch.int64) if tables else None
    announce(f"norm_rope weights={weights} tables={tables}")
    dev = [t if t is None else t.cuda() for t in (q, k, qw, kw, cos, sin, pos)]
    gq, gk = att.qk_norm_rope(*dev)
    _check(gq, q, qw, cos, sin, pos, False, "q")
    _check(gk, k, kw, cos, sin, pos, False, "k")


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("d", [64, 128])
def test_in_place_views_of_one_tensor(att, d, offset):
    """q, k and v side by side in one tensor (off the vectors' alignment too),
    rewritten where they are; v stays."""
    g = torch.Generator().manual_seed(5)
    hq, hkv, n = 6, 2, 37
    wide = (hq + 2 * hkv) * d + 8
    base = torch.randn(n * wide + 8, generator=g).half()
    dev = base.cuda()

    def views(t):
        r = t[offset:offset + n * wide].view(n, wide)
        return (r[:, :hq * d].view(n, hq, d), r[:, hq * d:(hq + hkv) * d].view(n, hkv, d),
                r[:, (hq + hkv) * d:])
    q, k, v = views(base)
    cos, sin = _tables(64, d)
    pos = torch.arange(n, dtype=torch.int32)
    qw, kw = torch.randn(d, generator=g).half(), torch.randn(d, generator=g).half()
    dq, dk, dv = views(dev)
    announce(f"norm_rope in place d={d} offset={offset}")
    att.qk_norm_rope_into(dq, dk, dq, dk, *(t.cuda() for t in (qw, kw, cos, sin, pos)))
    _check(dq, q, qw, cos, sin, pos, False, "q")
    _check(dk, k, kw, cos, sin, pos, False, "k")
    assert torch.equal(dv.cpu(), v)


def test_special_values(att):
    """Zeros, the type's largest values, NaN and Inf stay in their own head;
    positions out of the tables turn the rotated dims into NaN."""
    q = torch.randn(4, 3, 64, generator=torch.Generator().manual_seed(1))
    q[0, 0] = 0.0
    q[1, 1, 5] = float("inf")
    q[2, 2, 7] = float("nan")
    q[3, 0] = 1e30
    k = q[:, :1].clone()
    w = torch.ones(64)
    cos, sin = _tables(5, 32)
    pos = torch.tensor([0, 4, 1, 2], dtype=torch.int32)
    announce("norm_rope special values")
    gq, _ = att.qk_norm_rope(*(t.cuda() for t in (q, k, w, w, cos, sin, pos)))
    y, mag = norm_rope(q, w, cos, sin, pos, 1e-6, False)
    own = torch.zeros(4, 3, dtype=torch.bool)
    own[1, 1] = own[2, 2] = True
    own[3, 0] = True            # the squares overflow FP32: 0, as 1/sqrt(inf) is
    tol = norm_rope_tolerance(y, mag, torch.float32)
    assert_close(gq[~own.cuda()], y[~own].numpy(), tol[~own].numpy(), "others")
    assert bool(gq[2, 2].isnan().all())
    bad = torch.tensor([5, -1, 2 ** 31 - 1, 0], dtype=torch.int32)
    gq, _ = att.qk_norm_rope(*(t.cuda() for t in (q, k, w, w, cos, sin, bad)))
    assert bool(gq[:3, :, :32].isnan().all())
    assert bool(gq[0, :, 32:].isfinite().all()) and bool(gq[3, 1].isfinite().all())


def test_no_tokens_and_other_stream(att):
    q = torch.randn(0, 4, 64, device="cuda").half()
    w = torch.ones(64, device="cuda").half()
    gq, gk = att.qk_norm_rope(q, q, w, w)
    assert gq.shape == (0, 4, 64) and gk.shape == (0, 4, 64)
    q = torch.randn(33, 4, 64, device="cuda").half()
    want = att.qk_norm_rope(q, q, w, w)[0]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = att.qk_norm_rope(q, q, w, w)[0]
    s.synchronize()
    assert torch.equal(got, want)


def test_refusals(att):
    q = torch.randn(3, 4, 64, device="cuda").half()
    k = torch.randn(3, 2, 64, device="cuda").half()
    w = torch.ones(64, device="cuda").half()
    cos, sin = (t.cuda() for t in _tables(9, 64))
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")
    bad = [
        dict(k=k.float()), dict(k=k[:2]), dict(k=k.cpu()), dict(q=q[0]),
        dict(q=q.int(), k=k.int()), dict(q=q.transpose(1, 2)), dict(q_weight=w[:32]),
        dict(q_weight=w.int()), dict(q_weight=w.float()), dict(cos=None),
        dict(positions=None), dict(positions=pos[:2]), dict(positions=pos.float()),
        dict(cos=cos.half()), dict(cos=cos[:5]), dict(cos=cos.t().contiguous().t()),
        dict(cos=torch.zeros(9, 33, device="cuda"), sin=torch.zeros(9, 33, device="cuda")),
        dict(eps=float("nan")), dict(eps=-1.0),
        dict(q_weight=None, k_weight=None, cos=None, sin=None, positions=None)]
    for change in bad:
        args = dict(q=q, k=k, q_weight=w, k_weight=w, cos=cos, sin=sin, positions=pos)
        args.update(change)
        with pytest.raises(RuntimeError):
            att.qk_norm_rope(**args)
    rest = (w, w, cos, sin, pos)
    with pytest.raises(RuntimeError):            # shifted by a head: reads what is rewritten
        big = torch.randn(3, 5, 64, device="cuda").half()
        att.qk_norm_rope_into(big[:, :4], k, big[:, 1:], k.clone(), *rest)
    with pytest.raises(RuntimeError):            # both outputs in one place
        o = torch.empty_like(q)
        att.qk_norm_rope_into(q, q.clone(), o, o, *rest)
    with pytest.raises(RuntimeError):
        att.qk_norm_rope_into(q, k, q[:2], k, *rest)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("d,rot,shift", [(64, 64, 0), (128, 32, 0), (128, 128, 4), (256, 256, 0),
                                         (40, 24, 0), (512, 480, 0), (96, 96, 0), (160, 144, 0)])
def test_many_heads(att, dtype, inter, d, rot, shift):
    """Heads enough for groups of them, at odd counts, rows off 16 bytes too;
    every head as in a call of few, but for roundings (of FP32 16 each, of sums of
    two normed values, below 16 in all)."""
    g = torch.Generator(device="cuda").manual_seed(d)
    tokens, hq, hkv = 2117, 23, 8
    dt = DT[dtype]

    def rand(h):
        row = torch.randn(tokens, h * d + 8, generator=g, device="cuda").to(dt)
        return row[:, shift:shift + h * d].unflatten(1, (h, d))
    q, k = rand(hq), rand(hkv)
    qw, kw = ((1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(dt) for _ in range(2))
    cos, sin = (t.cuda() for t in _tables(50, rot))
    pos = torch.randint(0, 50, (tokens,), generator=g, dtype=torch.int32, device="cuda")
    announce(f"norm_rope many heads {dtype} inter={inter} d={d} rot={rot} shift={shift}")
    gq, gk = att.qk_norm_rope(q, k, qw, kw, cos, sin, pos, interleaved=inter)
    some = [0, 1, 777, tokens - 2, tokens - 1]
    for got, x, w, name in ((gq, q, qw, "q"), (gk, k, kw, "k")):
        _check(got[some], x[some].cpu(), w.cpu(), cos.cpu(), sin.cpu(), pos[some].cpu(), inter,
               name)
    few = 900                   # of few heads in all: one to a group
    for at in (0, tokens - few):
        part = slice(at, at + few)
        sq, sk = att.qk_norm_rope(q[part], k[part], qw, kw, cos, sin, pos[part],
                                  interleaved=inter)
        for a, b in ((gq[part], sq), (gk[part], sk)):
            assert bool(((a.double() - b.double()).abs()
                         <= 2 * UNIT[dt] * b.double().abs() + 2 * 16 * 2.0 ** -24 * 16).all())


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("tokens,hq,hkv,d,rot", [(2500, 13, 2, 128, 64), (901, 64, 9, 128, 128),
                                                 (5003, 7, 1, 256, 256), (20011, 3, 1, 64, 64),
                                                 (1501, 21, 3, 512, 512)])
def test_two_and_four_heads_to_a_group(att, dtype, tokens, hq, hkv, d, rot):
    """Between one head to a group and eight, at counts that leave groups short."""
    g = torch.Generator(device="cuda").manual_seed(tokens)
    dt = DT[dtype]
    q, k = (torch.randn(tokens, h, d, generator=g, device="cuda").to(dt) for h in (hq, hkv))
    qw, kw = ((1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(dt) for _ in range(2))
    cos, sin = (t.cuda() for t in _tables(50, rot))
    pos = torch.randint(0, 50, (tokens,), generator=g, dtype=torch.int32, device="cuda")
    announce(f"norm_rope some heads {dtype} {tokens}x({hq}+{hkv})x{d} rot={rot}")
    gq, gk = att.qk_norm_rope(q, k, qw, kw, cos, sin, pos)
    some = torch.linspace(0, tokens - 1, 24).long()
    for got, x, w, name in ((gq, q, qw, "q"), (gk, k, kw, "k")):
        _check(got[some], x[some].cpu(), w.cpu(), cos.cpu(), sin.cpu(), pos[some].cpu(), False,
               name)
