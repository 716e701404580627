"""A quantized paged key/value cache.  No counterpart in the reference (its
path ends at the projections).

Data format, per page of `page_size` tokens of every key/value head:

    k       int8  (pages, heads, page_size, D)              8 bits
            uint8 (pages, heads, page_size, D/2)            4 bits
    v       int8  (pages, heads, page_size/16, D, 16)       8 bits
            uint8 (pages, heads, page_size/16, D/2, 16)     4 bits
    scales  float32 (pages, heads, 2, page_size)            K's, then V's

With 4 bits byte j of a row holds dim 2j in its low nibble and 2j + 1 in its
high one, two's complement, as the INT4 weights do.  A value is its code times
the scale of its token and head.  V keeps 16 tokens of a dim side by side:
attention multiplies it over the tokens and reads them as one operand.

Quantization, per token and head, for K and V alike, with qmax 127 or 7, in
FP32 (every operation rounded once):

    scale = amax * fl(1 / qmax)
    code  = clamp(round_half_even(x * fl(1 / scale)), -qmax, qmax)

A vector whose amax is below 2^-100 gets scale 0 and codes 0; one with NaN or
Inf gets scale NaN, and every row of attention that sees it becomes NaN.

Which page holds a token: position p of sequence b is in page
block_table[b, p // page_size], at p % page_size.  The caller hands out pages.
"""
from __future__ import annotations

import torch

from . import _capi
from .ext import fast_module_or_none

HEAD_DIMS = (64, 128, 256)
PAGE_SIZES = (16, 32, 64, 128, 256)


def _fail(msg: str) -> None:
    raise RuntimeError(msg)


class KVCache:
    """The three tensors of a cache, checked once.  `KVCache.empty` makes one;
    the constructor takes tensors in the format above."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, scales: torch.Tensor):
        if k.dim() != 4 or v.dim() != 5 or scales.dim() != 4:
            _fail(f"a cache takes k of 4, v of 5 and scales of 4 dimensions, got "
                  f"{k.dim()}, {v.dim()} and {scales.dim()}")
        bits = {torch.int8: 8, torch.uint8: 4}.get(k.dtype)
        if bits is None or v.dtype != k.dtype:
            _fail(f"k and v must both be int8 (8 bits) or uint8 (4 bits), got {k.dtype} "
                  f"and {v.dtype}")
        if scales.dtype != torch.float32:
            _fail(f"scales must be float32, got {scales.dtype}")
        pages, heads, page, row = k.shape
        dim = row * 8 // bits
        if dim not in HEAD_DIMS:
            _fail(f"the head size must be one of {HEAD_DIMS}, got {dim}")
        if page not in PAGE_SIZES:
            _fail(f"the page size must be one of {PAGE_SIZES}, got {page}")
        if pages < 1 or not 1 <= heads <= 65535:
            _fail(f"a cache needs a page and 1 to 65535 heads, got {pages} pages of "
                  f"{heads} heads")
        if tuple(v.shape) != (pages, heads, page // 16, row, 16):
            _fail(f"v must be {(pages, heads, page // 16, row, 16)} for k "
                  f"{tuple(k.shape)}, got {tuple(v.shape)}")
        if tuple(scales.shape) != (pages, heads, 2, page):
            _fail(f"scales must be {(pages, heads, 2, page)} for k {tuple(k.shape)}, got "
                  f"{tuple(scales.shape)}")
        for name, t in (("k", k), ("v", v), ("scales", scales)):
            if not t.is_cuda:
                _fail(f"the cache's {name} must be a GPU tensor")
            if not t.is_contiguous():
                _fail(f"the cache's {name} must be contiguous")
            if t.device != k.device:
                _fail("the cache's tensors must be on one device")
            if t.data_ptr() % 16:
                _fail(f"the cache's {name} must be 16-byte aligned")
        self.k, self.v, self.scales = k, v, scales
        self.bits, self.pages, self.heads = bits, pages, heads
        self.head_dim, self.page_size = dim, page
        self.device = k.device
        self.c = _capi.CqKvCache(k.data_ptr(), v.data_ptr(), scales.data_ptr(), pages,
                                 heads, dim, page, bits)
        mod = fast_module_or_none()
        self.fast = mod and mod.Cache(k, v.data_ptr(), scales.data_ptr(), pages, heads, dim,
                                      page, bits)

    @classmethod
    def empty(cls, pages: int, heads: int, head_dim: int, page_size: int = 64,
              bits: int = 8, device: str = "cuda") -> "KVCache":
        """A cache of uninitialised pages: nothing reads a slot before `append`
        has written it, as long as lengths count written tokens only."""
        if bits not in (4, 8):
            _fail(f"bits must be 4 or 8, got {bits}")
        if head_dim not in HEAD_DIMS:
            _fail(f"the head size must be one of {HEAD_DIMS}, got {head_dim}")
        if page_size not in PAGE_SIZES:
            _fail(f"the page size must be one of {PAGE_SIZES}, got {page_size}")
        row = head_dim * bits // 8
        dt = torch.int8 if bits == 8 else torch.uint8
        return cls(torch.empty(pages, heads, page_size, row, dtype=dt, device=device),
                   torch.empty(pages, heads, page_size // 16, row, 16, dtype=dt,
                               device=device),
                   torch.empty(pages, heads, 2, page_size, dtype=torch.float32,
                               device=device))

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.scales))
