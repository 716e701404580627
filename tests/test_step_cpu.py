"""CPU tests of the operators of a step of many tokens: what the C entry points
refuse (the pointers here are never followed), and the test oracle."""
from __future__ import annotations

import ctypes

import pytest

from cudalab_amd import _capi
from step_oracle import place
from test_attention_cpu import BAD_CACHE, P, _cache

BAD = _capi.CQ_ERR_INVALID_ARG


def _place(**change):
    a = _capi.CqPlace(
        starts=P[0], counts=P[1], free_pages=P[2], taken_in=P[3], table=P[4], slots=P[5],
        positions=P[6], offsets=P[7], lengths=P[8], taken_out=P[9], table_stride=7, tokens=100,
        free_count=50, table_cols=5, batch=3, page_size=16)
    for n, v in change.items():
        setattr(a, n, v)
    return _capi.load().cq_place(ctypes.byref(a), None)


@pytest.mark.parametrize("change", [
    dict(batch=0), dict(batch=-1), dict(batch=2 ** 31 - 1), dict(tokens=-1), dict(tokens=2 ** 31),
    dict(page_size=8), dict(page_size=48), dict(page_size=512), dict(free_count=-1),
    dict(free_pages=None), dict(table=None), dict(table=P[4] + 2), dict(table_cols=0),
    dict(table_stride=4), dict(table_cols=2 ** 27, table_stride=2 ** 27),
    *(dict([(n, None)]) for n in ("starts", "counts", "offsets", "lengths", "taken_out", "slots",
                                  "positions")),
    *(dict([(n, P[12] + 2)]) for n in ("starts", "counts", "free_pages", "taken_in", "positions",
                                       "offsets", "lengths", "taken_out")),
    dict(slots=P[5] + 4), dict(taken_out=P[3]), dict(lengths=P[0]), dict(offsets=P[8] - 12),
    dict(positions=P[5] + 796), dict(table=P[0]), dict(free_pages=P[4] + 64),
    dict(counts=P[4] - 4, taken_in=P[4] + 72)])
def test_place_refuses(change):
    assert _place(**change) == BAD
    assert _capi.last_error()
    assert _capi.load().cq_place(None, None) == BAD


def _rows(cache=None, dtype=0, tokens=9, slots=P[5], k=P[6], v=P[7], strides=(256, 128, 256, 128)):
    c = cache or _cache()
    return _capi.load().cq_kv_append_rows(ctypes.byref(c), dtype, tokens, slots, k, strides[0],
                                          strides[1], v, strides[2], strides[3], None)


def test_append_rows_refuses():
    for change in BAD_CACHE:
        assert _rows(_cache(**change)) == BAD, change
    for change in (dict(dtype=3), dict(tokens=0), dict(tokens=-1), dict(tokens=2 ** 31),
                   dict(slots=None), dict(k=None), dict(v=None), dict(k=P[6] + 1),
                   dict(slots=P[5] + 4), dict(k=P[0]), dict(v=P[1] + 64), dict(slots=P[2]),
                   dict(strides=(-1, 128, 256, 128)), dict(strides=(256, 128, 256, 2 ** 41))):
        assert _rows(**change) == BAD, change
    # more workgroups than a launch holds
    assert _rows(_cache(heads=65535), tokens=2 ** 20) == BAD
    assert _capi.load().cq_kv_append_rows(None, 0, 1, P[5], P[6], 1, 1, P[7], 1, 1, None) == BAD


def test_place_by_hand():
    """Two sequences of 16-token pages: one of 15 tokens gets two, one of none
    gets three, of which the list holds two."""
    got = place([[4, 9, 9], [9, 9, 9]], [15, 0], [3, 18], 23, 16, [7, 5])
    assert got[0][:3] == [4 * 16 + 15, 7 * 16, 7 * 16 + 1]
    assert got[0][3:19] == [5 * 16 + i for i in range(16)]
    assert got[0][19:] == [-1] * 4
    assert got[1] == [15, 16, 17, *range(18), 0, 0]
    assert got[2:5] == ([0, 3, 21], [18, 18], 3)
    assert got[5] == [[4, 7, 9], [5, -1, 9]]


def _quantize(dtype=0, x=P[0], stride=64, tokens=5, k=64, codes=P[1], scales=P[2]):
    return _capi.load().cq_quantize_tokens(dtype, x, stride, tokens, k, codes, scales, None)


def _qgemm(workspace=False, **change):
    a = _capi.CqQgemm(x=P[0], x_scale=P[1], w=P[2], w_scale=P[3], out=P[4], x_stride=64,
                      tokens=5, n=7, k=64, workspace=P[5], workspace_bytes=1 << 31, dtype=0)
    for n, v in change.items():
        setattr(a, n, v)
    lib = _capi.load()
    return (lib.cq_qgemm_workspace(ctypes.byref(a)) if workspace
            else lib.cq_qgemm(ctypes.byref(a), None))


def test_qgemm_refuses():
    for change in (dict(dtype=3), dict(x=None), dict(codes=None), dict(scales=None), dict(x=P[0] + 1),
                   dict(scales=P[2] + 2), dict(stride=-1), dict(stride=2 ** 41), dict(tokens=0),
                   dict(tokens=2 ** 31 - 1), dict(k=0), dict(k=2 ** 31), dict(codes=P[0] + 8),
                   dict(scales=P[0]), dict(scales=P[1] + 4)):
        assert _quantize(**change) == BAD, change
    sizes = (dict(dtype=-1), dict(tokens=0), dict(tokens=2 ** 31 - 1), dict(n=0), dict(n=2 ** 31),
             dict(k=0), dict(k=131072, x_stride=131072), dict(x_stride=63),
             dict(x_stride=2 ** 41))
    for change in sizes:
        assert _qgemm(**change) == BAD, change
        assert _qgemm(True, **change) == -BAD, change
    for change in (*(dict([(n, None)]) for n in ("x", "x_scale", "w", "w_scale", "out")),
                   dict(x_scale=P[1] + 2), dict(w_scale=P[3] + 1), dict(out=P[4] + 8),
                   dict(out=P[0]), dict(out=P[2] + 432), dict(out=P[1]), dict(out=P[3] + 16)):
        assert _qgemm(**change) == BAD, change
    # more workgroups than a launch holds
    assert _qgemm(tokens=2 ** 31 - 512, n=2 ** 31 - 512) == BAD
    assert _capi.load().cq_qgemm(None, None) == BAD
    assert _capi.load().cq_qgemm_workspace(None) == -BAD


def _prompt(**change):
    a = _capi.CqPrompt(
        q=P[0], k=P[1], v=P[2], out=P[3], q_token_stride=512, q_head_stride=128,
        k_token_stride=256, k_head_stride=128, v_token_stride=256, v_head_stride=128,
        q_offsets=P[4], k_offsets=P[5], q_tokens=9, k_tokens=11, batch=2, q_heads=4, k_heads=2,
        head_dim=128, dtype=0, causal=1, softmax_scale=0.1)
    for n, v in change.items():
        setattr(a, n, v)
    return _capi.load().cq_prompt_attention(ctypes.byref(a), None)


@pytest.mark.parametrize("change", [
    *(dict([(n, None)]) for n in ("q", "k", "v", "out", "q_offsets")),
    *(dict([(n, P[12] + 8)]) for n in ("q", "k", "v", "out")), dict(q_offsets=P[4] + 2),
    dict(k_offsets=P[5] + 1), dict(batch=0), dict(batch=2 ** 31 - 1), dict(q_tokens=0),
    dict(q_tokens=2 ** 31 - 511), dict(k_tokens=-1), dict(k_tokens=2 ** 31 - 1), dict(q_heads=0),
    dict(q_heads=3), dict(k_heads=0), dict(q_heads=131072), dict(head_dim=96), dict(dtype=1),
    dict(dtype=3), dict(softmax_scale=float("nan")), dict(softmax_scale=float("inf")),
    dict(q_token_stride=-8), dict(q_head_stride=4), dict(k_token_stride=2 ** 24 + 8),
    dict(v_token_stride=2 ** 25), dict(v_head_stride=2 ** 41), dict(out=P[0]),
    dict(out=P[1] + 2048), dict(out=P[2] - 64), dict(out=P[4]), dict(out=P[5] - 9216 + 16)])
def test_prompt_refuses(change):
    assert _prompt(**change) == BAD
    assert _capi.last_error()
    assert _capi.load().cq_prompt_attention(None, None) == BAD


def test_prompt_refuses_too_many_workgroups():
    assert _prompt(batch=2 ** 30, q_heads=65534) == BAD


def test_tree_refuses():
    a = _capi.CqAttention(
        q=P[6], out=P[7], q_batch_stride=5120, q_token_stride=1024, q_head_stride=128,
        table=P[3], lengths=P[4], counts=None, prefix_table=None, table_stride=5,
        workspace=P[9], workspace_bytes=1 << 31, table_cols=5, prefix_cols=0, prefix_len=0,
        batch=2, tokens=5, q_heads=8, dtype=0, softmax_scale=0.1)
    c, lib = _cache(), _capi.load()

    def call(seen=P[10], cache=c, args=a):
        return lib.cq_attention_tree(cache and ctypes.byref(cache), args and ctypes.byref(args),
                                     seen, None)

    for bad in (dict(seen=None), dict(seen=P[10] + 4), dict(seen=P[7] + 64), dict(seen=P[9]),
                dict(cache=None), dict(args=None), dict(cache=_cache(head_dim=96))):
        assert call(**bad) == BAD, bad
    a.q = P[6] + 8
    assert call() == BAD
    a.q, a.workspace_bytes = P[6], 16
    assert call() == _capi.CQ_ERR_BUFFER_TOO_SMALL
