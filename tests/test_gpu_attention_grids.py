"""GPU tests of calls around attention of more workgroups than one launch
takes (HIP counts a launch's threads in 32 bits)."""
from __future__ import annotations

import pytest
import torch

from attention_oracle import Pages, assert_close, norm_rope, norm_rope_tolerance, quantize
from conftest import announce

pytestmark = pytest.mark.gpu
MANY = 2 ** 24 + 37              # workgroups of 256 threads: 2^32 threads and more


@pytest.fixture(scope="module")
def att(cuda):
    from cudalab_amd.build import build
    return build("attention")


@pytest.mark.parametrize("bits", [8, 4])
def test_cache(att, bits):
    """One token of each of very many sequences, a few of which have a page."""
    page, dim, some = 16, 64, [0, 5, 2 ** 24 - 1, 2 ** 24, MANY - 1]
    pages = Pages(len(some), 1, dim, page, bits)
    cache = pages.device()
    table = torch.full((MANY, 1), -1, dtype=torch.int32, device="cuda")
    starts = torch.zeros(MANY, dtype=torch.int32, device="cuda")
    x = torch.randn(1, 1, 1, dim, generator=torch.Generator().manual_seed(bits)).half()
    codes, scale = quantize(x.float().numpy()[0, 0], bits)
    for i, b in enumerate(some):
        table[b], starts[b] = i, 3 + i
        for which in (0, 1):
            pages.put(i, 3 + i, which, codes, scale)
    many = x.cuda().expand(MANY, 1, 1, dim)
    announce(f"append to {MANY} sequences, {bits} bits")
    att.append(cache, many, many, table, starts)
    k, v, s = pages.tensors()
    for got, want in ((cache.k, k), (cache.v, v), (cache.scales, s)):
        assert torch.equal(got.cpu(), want)
    announce(f"read of {MANY} sequences, {bits} bits")
    gk, gv = att.read(cache, table, starts, None, 1)
    want = torch.from_numpy(codes.astype("f4") * scale[..., None]).half().view(dim)
    for got in (gk, gv):
        assert all(torch.equal(got[b].cpu().view(dim), want) for b in some)
        assert int(got.any(3).sum()) == len(some)


def test_norm_rope(att):
    """Heads that take the element kernel, four to a workgroup."""
    tokens, hq, hkv, d = 2 ** 20, 64, 1, 2
    assert tokens * (hq + hkv) > 4 * MANY
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k = (torch.rand(tokens, h, d, generator=g, device="cuda").half() + 0.5 for h in (hq, hkv))
    w = torch.rand(d, generator=g, device="cuda").half() + 0.5
    ang = torch.rand(9, d // 2, generator=g, device="cuda")
    pos = torch.randint(0, 9, (tokens,), generator=g, dtype=torch.int32, device="cuda")
    announce(f"norm_rope of {tokens * (hq + hkv)} heads of {d}")
    out = att.qk_norm_rope(q, k, w, w, ang.cos(), ang.sin(), pos)
    edge = 2 ** 26 // (hq + hkv)
    some = [0, edge - 1, edge, edge + 1, tokens - 1]
    for got, x in zip(out, (q, k)):
        y, mag = norm_rope(x[some].cpu(), w.cpu(), ang.cos().cpu(), ang.sin().cpu(),
                           pos[some].cpu(), 1e-6, False)
        tol = norm_rope_tolerance(y, mag, x.dtype)
        assert_close(got[some], y.numpy(), tol.numpy(), "heads")
        # a rotated, normed pair has the weights' size: nowhere left out
        size = got.float().square().sum(-1)
        assert bool(((size > 0.2) & (size < 4.6)).all())


def test_join(att):
    """Rows that are joined four to a workgroup."""
    from cudalab_amd.kvcache import KVCache
    group, dim = 32, 64
    batch = 4 * MANY // group + 1
    cache = KVCache.empty(1, 1, dim, 16, 8)
    for t in (cache.k, cache.v):
        t.zero_()
    cache.scales.fill_(0.5)
    cache.v[0, 0, 0, :, 0] = torch.arange(dim, device="cuda").to(torch.int8)
    q = torch.ones(1, 1, group, dim, device="cuda").half().expand(batch, 1, group, dim)
    table = torch.zeros(batch, 1, dtype=torch.int32, device="cuda")
    lengths = torch.ones(batch, dtype=torch.int32, device="cuda")
    lengths[7::1000] = 0
    announce(f"attention of {batch * group} rows")
    out = att.forward(q, cache, table, lengths)
    want = (torch.arange(dim, device="cuda") * 0.5).half()
    for at in range(0, batch, 1 << 18):
        part = out[at:at + (1 << 18)]
        live = lengths[at:at + (1 << 18)].bool()[:, None, None, None]
        assert torch.equal(part, torch.where(live, want, want.new_zeros(())).expand_as(part)), at
