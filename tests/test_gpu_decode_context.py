"""GPU tests of the decode step with a context: norms, the quantized cache and
attention between the projections."""
from __future__ import annotations

import pytest
import torch

from attention_oracle import Pages, assert_close, attention, norm_rope, norm_rope_tolerance
from conftest import announce

pytestmark = pytest.mark.gpu

SIZES = dict(hidden=1024, inter=2048)


def _model(bits, kv, context=150, layers=2, room=4):
    from cudalab_amd.decode import DecodeModel
    return DecodeModel("int4gemv", layers=layers, seed=11, kv=kv, context=context,
                       cache_bits=bits, room=room, **SIZES)


def _pages_of(cache):
    """The host's view of a cache on the device."""
    page = Pages(cache.pages, cache.heads, cache.head_dim, cache.page_size, cache.bits)
    k, v = cache.k.cpu().int(), cache.v.cpu().int()
    p, h, n, row, _ = v.shape
    v = v.swapaxes(3, 4).reshape(p, h, n * 16, row)
    if cache.bits == 4:
        k, v = (torch.stack((t & 15, t >> 4), -1).flatten(-2) for t in (k, v))
        k, v = (t - ((t & 8) << 1) for t in (k, v))
    page.k, page.v, page.scales = k.numpy(), v.numpy(), cache.scales.cpu().numpy()
    return page


def _results(m):
    return m.outputs() + [L.out["o_in"].clone() for L in m.layers]


@pytest.mark.parametrize("bits,kv", [(8, 256), (4, 256), (8, 1024)])
def test_layer_against_the_formula(cuda, bits, kv):
    """The first layer's rotated q and k, its cached token and o's input."""
    m = _model(bits, kv)
    L = m.layers[0]
    announce(f"decode with a context, {bits} bits, kv {kv}")
    raw = {n: m.ext.forward(m.variant, *L.w[n], m.x0).view(1, -1, 128) for n in ("q", "k", "v")}
    m.step_grouped()
    torch.cuda.synchronize()
    at = m.context
    for n, w in zip(("q", "k"), L.norm):
        want, mag = norm_rope(raw[n], w, m.cos, m.sin, m.position.cpu(), 1e-6, False)
        tol = norm_rope_tolerance(want, mag, torch.float16)
        assert_close(L.out[n].view(1, -1, 128), want.numpy(), tol.numpy(), n)
    k, v = m.att.read(L.cache, m.table, m.position, None, 1, torch.float32)
    top = 127 if bits == 8 else 7
    for got, x in ((k, L.out["k"]), (v, raw["v"])):
        x = x.view(-1, 128).float()
        step = x.abs().amax(1, keepdim=True) / top
        assert bool(((got.view(-1, 128) - x).abs() <= 0.501 * step).all())
    table = [m.table[0].tolist()]
    want, tol = attention(L.out["q"].view(1, 1, -1, 128), _pages_of(L.cache), table, [at + 1])
    assert_close(L.out["o_in"].view(1, 1, -1, 128), want, tol, "o's input")


@pytest.mark.parametrize("bits,kv", [(8, 256), (4, 1024)])
def test_modes_bit_identical_over_tokens(cuda, bits, kv):
    """Sequential, grouped and replayed steps, token after token."""
    a, b, c = (_model(bits, kv) for _ in range(3))
    graph = c.capture()
    for i in range(4):
        announce(f"decode with a context, {bits} bits, token {i}")
        a.step_sequential()
        b.step_grouped()
        graph.replay()
        torch.cuda.synchronize()
        ref = _results(a)
        assert all(bool(torch.isfinite(t).all()) for t in ref)
        for m in (b, c):
            for x, y in zip(ref, _results(m)):
                assert torch.equal(x, y), i
        for m in (a, b, c):
            m.advance()
        torch.cuda.synchronize()
    assert int(a.length) == a.context + 5


def test_run_reports_the_context(cuda):
    from cudalab_amd import decode
    announce("decode run with a context")
    res = decode.run(layers=1, steps=2, warmup=1, model="70b", context=100, cache_bits=4)
    assert res["context"] == 100 and res["cache_bits"] == 4
    assert res["launches_per_layer"]["graph"] == 8
    assert res["cache_bytes_per_step"] == 101 * 8 * 2 * (64 + 4)
    assert all(res[m]["us_per_step"] > 0 for m in decode.MODES)
