"""GPU tests of what attention takes as it is: queries at any address and of
any stride that torch gives a single row, and which errors other arguments
raise."""
from __future__ import annotations

import pytest
import torch

from conftest import announce
from test_gpu_attention import _ints, _q, _setup, att  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("off", [1, 4, 7])
def test_contiguous_queries_at_any_address(att, off):                # noqa: F811
    """A contiguous q off the 16 bytes that the kernels read at once."""
    lens = [130, 20]
    pages, table, _ = _setup(lens, 2, 64, 16, 8)
    q = _q(2, 3, 4, 64, "fp16").cuda()
    moved = torch.empty(q.numel() + 8, dtype=q.dtype, device="cuda")[off:off + q.numel()]
    moved = moved.view(q.shape).copy_(q)
    assert moved.is_contiguous() and moved.data_ptr() % 16
    cache, tab, ln = pages.device(), _ints(table), _ints(lens)
    announce(f"attention contiguous q {off} elements off")
    assert torch.equal(att.forward(moved, cache, tab, ln), att.forward(q, cache, tab, ln))


def test_strides_of_single_rows(att):                                # noqa: F811
    """A dimension of one row may have any stride."""
    pages, table, _ = _setup([50], 1, 64, 16, 8)
    cache, tab, ln = pages.device(), _ints(table), _ints([50])
    q = _q(1, 1, 1, 64, "fp16").cuda()
    want = att.forward(q, cache, tab, ln)
    announce("attention strides of single rows")
    for strides in ((67, 67, 67, 1), (1, 1, 1, 1), (64, 3, 64, 1)):
        view = torch.as_strided(q, q.shape, strides)
        assert torch.equal(att.forward(view, cache, tab, ln), want), strides


def test_wrong_types_raise_runtime_error(att):                       # noqa: F811
    from cudalab_amd.kvcache import KVCache
    c = KVCache.empty(4, 2, 64, 16, 8)
    q = torch.zeros(2, 3, 4, 64, device="cuda").half()
    good = dict(q=q, cache=c, block_table=_ints([[0], [1]]), lengths=_ints([3, 3]))
    pages = _ints([2])
    announce("attention arguments of wrong types")
    for change in (dict(prefix=pages), dict(prefix=3), dict(prefix=(pages,)),
                   dict(prefix=(pages, 1, 2)), dict(prefix="ab"), dict(prefix=(None, 3)),
                   dict(prefix=(pages, True)), dict(prefix=(pages, "3")), dict(scale="1"),
                   dict(scale=[1.0]), dict(scale=1e60), dict(scale=10 ** 400)):
        with pytest.raises(RuntimeError):
            att.forward(**{**good, **change})
        with pytest.raises(RuntimeError):
            att.forward_into(out=torch.empty_like(q), **{**good, **change})
    k = torch.zeros(3, 2, 64, device="cuda").half()
    w = torch.ones(64, device="cuda").half()
    for eps in ("1", None, [1e-6], 10 ** 400):
        with pytest.raises(RuntimeError):
            att.qk_norm_rope(k, k, w, w, eps=eps)
        with pytest.raises(RuntimeError):
            att.qk_norm_rope_into(k, k, torch.empty_like(k), torch.empty_like(k), w, w, eps=eps)
