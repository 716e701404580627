"""CPU tests of the operators around attention: what the C entry points and the
Python layer refuse (the pointers here are never followed), and the test
oracle's own definitions."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from attention_oracle import Pages, attention, norm_rope, quantize
from cudalab_amd import _capi

P = [0x100000000 * (i + 1) for i in range(16)]


def _norm_rope(**change):
    a = _capi.CqNormRope(
        q=P[0], k=P[1], q_out=P[2], k_out=P[3], q_token_stride=512, q_head_stride=128,
        k_token_stride=256, k_head_stride=128, q_out_token_stride=512, q_out_head_stride=128,
        k_out_token_stride=256, k_out_head_stride=128, q_weight=P[4], k_weight=P[5],
        cos_table=P[6], sin_table=P[7], positions=P[8], tokens=3, table_rows=9, q_heads=4,
        k_heads=2, head_dim=128, rot_dim=128, dtype=0, weight_dtype=0, positions_64=0,
        interleaved=0, eps=1e-6)
    for n, v in change.items():
        setattr(a, n, v)
    return _capi.load().cq_qk_norm_rope(ctypes.byref(a), None)


@pytest.mark.parametrize("change", [
    dict(q=None), dict(k_out=None), dict(q=P[0] + 1), dict(k_weight=P[5] + 1), dict(tokens=0),
    dict(tokens=-1), dict(tokens=2 ** 31), dict(q_heads=-1), dict(q_heads=0, k_heads=0),
    dict(q_heads=65535), dict(head_dim=0), dict(head_dim=127), dict(head_dim=1026),
    dict(dtype=3), dict(weight_dtype=-1), dict(q_token_stride=-1), dict(k_head_stride=-8),
    dict(cos_table=None), dict(sin_table=None), dict(rot_dim=130), dict(rot_dim=0),
    dict(rot_dim=7), dict(positions=None), dict(positions=P[8] + 2),
    dict(positions=P[8] + 4, positions_64=1), dict(table_rows=0), dict(cos_table=P[6] + 2),
    dict(eps=-1.0), dict(eps=math.inf), dict(eps=math.nan),
    dict(q_weight=None, k_weight=None, cos_table=None, sin_table=None),
    dict(q_out=P[0] + 256), dict(q_out=P[1]), dict(k_out=P[0]), dict(k_out=P[2]),
    dict(q_out=P[4] - 16), dict(k_out=P[6]), dict(q_out=P[8] - 512),
    dict(q_out=P[0], q_out_token_stride=1024),           # in place with another stride
    dict(q_out_head_stride=64), dict(k_out_token_stride=128),
    # q and k side by side, k's heads reaching into the next token's q
    dict(q=P[0], q_out=P[0], k=P[0] + 1024, k_out=P[0] + 1024, k_token_stride=512,
         k_out_token_stride=512)])
def test_norm_rope_refuses(change):
    assert _norm_rope(**change) == _capi.CQ_ERR_INVALID_ARG
    assert _capi.last_error()


def _cache(**change):
    c = _capi.CqKvCache(P[0], P[1], P[2], 8, 2, 128, 64, 8)
    for n, v in change.items():
        setattr(c, n, v)
    return c


def _slots(**change):
    s = _capi.CqKvSlots(P[3], P[4], P[5], 5, 5, 3, 7)
    for n, v in change.items():
        setattr(s, n, v)
    return s


BAD_CACHE = [dict(k=None), dict(v=None), dict(scales=None), dict(k=P[0] + 8),
             dict(scales=P[2] + 4), dict(pages=0), dict(pages=2 ** 31), dict(heads=0),
             dict(heads=65536), dict(head_dim=96), dict(page_size=8), dict(page_size=48),
             dict(page_size=512), dict(bits=5)]
BAD_SLOTS = [dict(table=None), dict(starts=None), dict(table=P[3] + 2), dict(starts=P[4] + 1),
             dict(counts=P[5] + 1), dict(table_stride=4), dict(table_cols=0), dict(batch=0),
             dict(tokens=0), dict(tokens=-4)]


def _append(c, s, dtype=0, k=P[6], v=P[7], stride=256):
    n = stride
    return _capi.load().cq_kv_append(ctypes.byref(c), ctypes.byref(s), dtype, k, 7 * n, n, 128,
                                     v, 7 * n, n, 128, None)


def _read(c, s, dtype=0, k=P[6], v=P[7]):
    return _capi.load().cq_kv_read(ctypes.byref(c), ctypes.byref(s), dtype, k, v, None)


@pytest.mark.parametrize("call", [_append, _read])
def test_cache_calls_refuse(call):
    bad = _capi.CQ_ERR_INVALID_ARG
    for change in BAD_CACHE:
        assert call(_cache(**change), _slots()) == bad, change
    for change in BAD_SLOTS:
        assert call(_cache(), _slots(**change)) == bad, change
    for change in (dict(dtype=3), dict(k=None), dict(v=None), dict(k=P[6] + 1), dict(k=P[0]),
                   dict(v=P[1] + 64), dict(k=P[2])):
        assert call(_cache(), _slots(), **change) == bad, change
    # more workgroups than a launch holds
    assert call(_cache(heads=65535), _slots(batch=2 ** 20, tokens=1)) == bad


def test_cache_calls_refuse_overlaps():
    bad = _capi.CQ_ERR_INVALID_ARG
    assert _append(_cache(v=P[0] + 1024), _slots()) == bad
    assert _append(_cache(), _slots(), stride=-1) == bad
    assert _append(_cache(), _slots(table=P[0])) == bad
    assert _read(_cache(), _slots(), k=P[6], v=P[6] + 1024) == bad
    assert _read(_cache(), _slots(), k=P[4]) == bad
    assert _read(_cache(), _slots(), k=P[3] - 32) == bad


def _attention(cache=None, workspace=False, **change):
    a = _capi.CqAttention(
        q=P[6], out=P[7], q_batch_stride=1024, q_token_stride=1024, q_head_stride=128,
        table=P[3], lengths=P[4], counts=None, prefix_table=P[5], table_stride=5,
        workspace=P[9], workspace_bytes=1 << 31, table_cols=5, prefix_cols=3, prefix_len=150,
        batch=2, tokens=1, q_heads=8, dtype=0, softmax_scale=0.1)
    for n, v in change.items():
        setattr(a, n, v)
    c = cache or _cache()
    lib = _capi.load()
    if workspace:
        return lib.cq_attention_workspace(ctypes.byref(c), ctypes.byref(a))
    return lib.cq_attention(ctypes.byref(c), ctypes.byref(a), None)


SHAPES = [dict(batch=0), dict(tokens=0), dict(q_heads=0), dict(q_heads=7), dict(q_heads=65536),
          dict(batch=2 ** 20, tokens=2 ** 20), dict(dtype=1), dict(prefix_len=-1),
          dict(prefix_len=193), dict(prefix_cols=0), dict(table_cols=0),
          dict(softmax_scale=math.nan), dict(softmax_scale=-math.inf)]


def test_attention_refuses():
    bad = _capi.CQ_ERR_INVALID_ARG
    for change in BAD_CACHE:
        assert _attention(_cache(**change)) == bad, change
        assert _attention(_cache(**change), workspace=True) == -bad, change
    for change in SHAPES:
        assert _attention(**change) == bad, change
        assert _attention(workspace=True, **change) == -bad, change
    for change in (dict(q=None), dict(out=None), dict(table=None), dict(lengths=None),
                   dict(prefix_table=None), dict(q=P[6] + 8), dict(out=P[7] + 2),
                   dict(lengths=P[4] + 2), dict(prefix_table=P[5] + 1), dict(counts=P[8] + 1),
                   dict(table_stride=3), dict(q_head_stride=132), dict(q_batch_stride=-8),
                   dict(out=P[6]), dict(out=P[0] + 64), dict(out=P[4] - 16), dict(out=P[2])):
        assert _attention(**change) == bad, change
    assert _attention(workspace=True) >= 0
    lib = _capi.load()
    assert lib.cq_attention(None, None, None) == bad
    assert lib.cq_attention_workspace(None, None) == -bad
    assert lib.cq_qk_norm_rope(None, None) == bad
    assert lib.cq_kv_append(None, None, 0, None, 0, 0, 0, None, 0, 0, 0, None) == bad
    assert lib.cq_kv_read(None, None, 0, None, None, None) == bad


def test_python_layer_refuses_host_tensors():
    from cudalab_amd.build import build
    from cudalab_amd.kvcache import KVCache
    att = build("attention")
    assert att is build("attention")
    x = torch.zeros(2, 4, 64).half()
    with pytest.raises(RuntimeError, match="GPU tensor"):
        att.qk_norm_rope(x, x, x[0, 0], x[0, 0])
    with pytest.raises(RuntimeError, match="GPU tensor"):
        KVCache(torch.zeros(1, 1, 16, 64, dtype=torch.int8),
                torch.zeros(1, 1, 1, 64, 16, dtype=torch.int8), torch.zeros(1, 1, 2, 16))
    with pytest.raises(RuntimeError, match="KVCache"):
        att.append(None, x, x, x, x)
    with pytest.raises(RuntimeError, match="KVCache"):
        att.forward(x, None, x, x)


# ----------------------------------------------------- the oracle's own sense
def test_oracle_quantizer():
    x = np.array([[0, 127, -63.5, 0.5, 1.5], [0] * 5, [np.nan, 1, 2, 3, 4]], np.float32)
    codes, scale = quantize(x, 8)
    assert codes[0].tolist() == [0, 127, -64, 0, 2] and scale[0] == np.float32(1)
    assert not codes[1].any() and scale[1] == 0
    assert not codes[2].any() and np.isnan(scale[2])
    codes, scale = quantize(np.array([[7.0, -7.0, 3.4]], np.float32), 4)
    assert codes[0].tolist() == [7, -7, 3]


def test_oracle_layout_and_attention():
    pages = Pages(3, 2, 64, 16, 4, seed=1)
    k, v, _ = pages.tensors()
    assert k.shape == (3, 2, 16, 32) and v.shape == (3, 2, 1, 32, 16)
    for p, h, t, d in ((0, 0, 0, 0), (2, 1, 13, 63), (1, 0, 5, 30)):
        for byte, code in ((k[p, h, t, d // 2], pages.k[p, h, t, d]),
                           (v[p, h, 0, d // 2, t], pages.v[p, h, t, d])):
            nib = (int(byte) >> (4 * (d % 2))) & 15
            assert (nib ^ 8) - 8 == code
    table = [[2, 0], [1, -1]]
    q = torch.randn(2, 3, 4, 64, dtype=torch.float64).half()
    out, tol = attention(q, pages, table, [20, 2])
    kk, _ = pages.values(table[0], 0, 20, 0)
    vv, _ = pages.values(table[0], 0, 20, 1)
    s = kk[1, :19] @ q[0, 1, 3].double().numpy() / 8
    p = np.exp(s - s.max())
    assert np.allclose(out[0, 1, 3], (p / p.sum()) @ vv[1, :19])
    assert (out[1, 0] == 0).all() and (out[1, 1:] != 0).any() and (tol >= 0).all()


def test_oracle_rotation_turns():
    """A rotation by an angle and by its negative give the input back, in both
    styles, and lengths of pairs stay."""
    x = torch.randn(2, 3, 64, dtype=torch.float64)
    ang = torch.rand(4, 16) * 6
    pos = torch.tensor([1, 3])
    for inter in (False, True):
        y, _ = norm_rope(x, None, ang.cos(), ang.sin(), pos, 1e-6, inter)
        assert not torch.allclose(x[..., :32], y[..., :32]) and torch.equal(x[..., 32:], y[..., 32:])
        z, _ = norm_rope(y, None, ang.cos(), -ang.sin(), pos, 1e-6, inter)
        assert torch.allclose(x, z, atol=1e-6)


def test_attention_refuses_more_keys_than_ints_count():
    """Tables whose positions, or whose tiles over all units, pass 31 bits."""
    bad = _capi.CQ_ERR_INVALID_ARG
    one = dict(batch=1, q_heads=_cache().heads, prefix_len=0)
    page = _cache().page_size
    assert _attention(workspace=True, table_cols=2 ** 30 // page, **one) >= 0
    for change in (dict(table_cols=2 ** 31 // page), dict(table_cols=2 ** 30),
                   dict(table_cols=2 ** 30 // page, batch=2 ** 10)):
        assert _attention(**{**one, **change}) == bad, change
        assert _attention(workspace=True, **{**one, **change}) == -bad, change
