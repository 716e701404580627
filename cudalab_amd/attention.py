"""The operators between a decoder's q/k/v projections and its o projection,
over the C ABI: `build("attention")` returns the one `AttentionExt`.  No
counterpart in the reference, whose path ends at the projections.

    att = build("attention")
    q, k = att.qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions)
    att.append(cache, k, v, block_table, lengths_before)
    out = att.forward(q, cache, block_table, lengths_after)

and, for prompts whose tokens lie end to end ("packed"),

    p = att.place(block_table, starts, counts, tokens, page_size, free_pages)
    q, k = att.qk_norm_rope(q, k, q_weight, k_weight, cos, sin, p.positions)
    att.append_rows(cache, k, v, p.slots)
    out = att.prompt(q, k, v, p.offsets)

Every check that needs only shapes, types and devices runs on the host before
anything is launched and raises RuntimeError.  Lengths, positions and page
numbers live on the device and are never read by the host: the kernels check
them against the tensors' sizes (a token outside them is not written, reads as
zeros and is not attended to).  Launches go on the current torch stream of the
tensors' device, work inside a HIP graph, and keep nothing between calls.

Each call is first offered to the fast path (csrc/cq_pyattn.h): one C++ call
that applies the same rules to the tensors' metadata and makes the library
call.  It launches nothing for a call it does not accept, and the checked path
here then runs and raises.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _capi
from .ext import _on_device, fast_module_or_none
from .kvcache import HEAD_DIMS, PAGE_SIZES, KVCache

_DTYPES = {torch.float16: _capi.CQ_DTYPE_F16, torch.float32: _capi.CQ_DTYPE_F32,
           torch.bfloat16: _capi.CQ_DTYPE_BF16}


def _fail(msg: str) -> None:
    raise RuntimeError(msg)


def _check(status: int, what: str) -> None:
    if status != _capi.CQ_OK:
        _fail(f"{what} failed (status {status}): {_capi.last_error()}")


def _gpu(name: str, t: torch.Tensor, device: torch.device) -> None:
    if not isinstance(t, torch.Tensor):
        _fail(f"{name} must be a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        _fail(f"{name} must be a GPU tensor")
    if t.device != device:
        _fail(f"{name} must be on {device}, got {t.device}")


def _heads(name: str, t: torch.Tensor, dims: int, device: torch.device) -> None:
    """A tensor of heads: `dims` dimensions, the last contiguous."""
    _gpu(name, t, device)
    if t.dim() != dims:
        _fail(f"{name} must have {dims} dimensions, got {t.dim()}")
    if t.dtype not in _DTYPES:
        _fail(f"{name} must be float16, bfloat16 or float32, got {t.dtype}")
    if t.size(-1) > 1 and t.stride(-1) != 1:
        _fail(f"the last dimension of {name} must be contiguous")


def _ints(name: str, t: torch.Tensor, shape: tuple, device: torch.device) -> None:
    _gpu(name, t, device)
    if t.dtype != torch.int32:
        _fail(f"{name} must be int32, got {t.dtype}")
    if tuple(t.shape) != shape:
        _fail(f"{name} must be of shape {shape}, got {tuple(t.shape)}")
    if not t.is_contiguous():
        _fail(f"{name} must be contiguous")


def _table(name: str, t: torch.Tensor, batch: int, device: torch.device) -> None:
    _gpu(name, t, device)
    if t.dtype != torch.int32:
        _fail(f"{name} must be int32, got {t.dtype}")
    if t.dim() != 2 or t.size(0) != batch or t.size(1) < 1:
        _fail(f"{name} must be ({batch}, pages), got {tuple(t.shape)}")
    if t.size(1) > 1 and t.stride(1) != 1:
        _fail(f"the rows of {name} must be contiguous")


def _count(name: str, n) -> int:
    if isinstance(n, bool) or not isinstance(n, int) or not 0 <= n < 2 ** 31:
        _fail(f"{name} must be an int in [0, 2^31), got {n!r}")
    return n


def _number(name: str, x) -> float:
    try:
        if hasattr(x, "__float__"):
            return float(x)
    except (TypeError, ValueError, OverflowError):
        pass
    _fail(f"{name} must be a number that a float holds, got {type(x).__name__}")


def _pair(prefix) -> tuple:
    if not isinstance(prefix, (tuple, list)) or len(prefix) != 2:
        _fail(f"prefix must be a pair (pages, length), got {type(prefix).__name__}")
    return prefix


class Placed(NamedTuple):
    """Where a packed batch's tokens go (AttentionExt.place)."""
    slots: torch.Tensor        # int64 (tokens,): page * page_size + offset, or -1
    positions: torch.Tensor    # int32 (tokens,)
    offsets: torch.Tensor      # int32 (batch + 1,): rows before each sequence
    lengths: torch.Tensor      # int32 (batch,): tokens with the added ones
    taken: torch.Tensor        # int32 (1,): entries of the free list that are gone


class PlacedHeld(NamedTuple):
    """Placed, and the pages that each sequence holds then (place with `held`)."""
    slots: torch.Tensor
    positions: torch.Tensor
    offsets: torch.Tensor
    lengths: torch.Tensor
    taken: torch.Tensor
    held: torch.Tensor         # int32 (batch,)


class AttentionExt:
    """Norms with rotation, the quantized cache and attention over it."""

    def __init__(self) -> None:
        self._lib = _capi.load()
        mod = fast_module_or_none()
        self._fast = mod and mod.AttentionCalls(*(_capi.entry_address(n) for n in (
            "cq_qk_norm_rope", "cq_kv_append", "cq_kv_read", "cq_attention",
            "cq_attention_workspace", "cq_attention_tree", "cq_attention_tree_workspace",
            "cq_last_error")))
        self._step = mod and mod.StepCalls(*(_capi.entry_address(n) for n in (
            "cq_place", "cq_place_held", "cq_kv_append_rows", "cq_prompt_attention", "cq_last_error")))

    # ---- norms and rotation ----
    def qk_norm_rope(self, q: torch.Tensor, k: torch.Tensor,
                     q_weight: Optional[torch.Tensor] = None,
                     k_weight: Optional[torch.Tensor] = None,
                     cos: Optional[torch.Tensor] = None,
                     sin: Optional[torch.Tensor] = None,
                     positions: Optional[torch.Tensor] = None, *, eps: float = 1e-6,
                     interleaved: bool = False
                     ) -> tuple[torch.Tensor, torch.Tensor]:
        """RMS norm of each head of q (tokens, Hq, D) and k (tokens, Hkv, D),
        then the rotation of its first R dims, into new contiguous tensors.
        See qk_norm_rope_into."""
        eps, interleaved = _number("eps", eps), bool(interleaved)
        if self._fast is not None:
            got = self._fast.norm_rope(q, k, None, None, q_weight, k_weight, cos, sin,
                                       positions, eps, interleaved)
            if got is not None:
                return got
        for name, t in (("q", q), ("k", k)):
            if not isinstance(t, torch.Tensor):
                _fail(f"{name} must be a tensor, got {type(t).__name__}")
        qo = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        ko = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        self._norm_rope(q, k, qo, ko, q_weight, k_weight, cos, sin, positions, eps,
                        interleaved)
        return qo, ko

    def qk_norm_rope_into(self, q, k, q_out, k_out, q_weight=None, k_weight=None,
                          cos=None, sin=None, positions=None, *, eps: float = 1e-6,
                          interleaved: bool = False) -> None:
        """qk_norm_rope into given tensors; q_out may be q and k_out may be k.

        In FP32, rounded once to q's type:
            n  = x * weight / sqrt(mean(x^2) + eps)     weight None: n = x
            a' = a cos - b sin, b' = b cos + a sin       cos None: no rotation
        for the pairs (a, b) = (n[i], n[i + R/2]), or (n[2i], n[2i + 1]) if
        `interleaved`, with cos, sin float32 (rows, R/2) taken at the token's
        row positions[token] (int32 or int64).  Tokens and heads may have any
        stride; a position outside the tables turns the token's rotated dims
        into NaN."""
        eps, interleaved = _number("eps", eps), bool(interleaved)
        if self._fast is not None and q_out is not None and k_out is not None \
                and self._fast.norm_rope(q, k, q_out, k_out, q_weight, k_weight, cos, sin,
                                         positions, eps, interleaved) is not None:
            return
        self._norm_rope(q, k, q_out, k_out, q_weight, k_weight, cos, sin, positions, eps,
                        interleaved)

    def _norm_rope(self, q, k, q_out, k_out, q_weight, k_weight, cos, sin, positions, eps,
                   interleaved) -> None:
        if not isinstance(q, torch.Tensor):
            _fail(f"q must be a tensor, got {type(q).__name__}")
        dev = q.device
        for name, t in (("q", q), ("k", k), ("q_out", q_out), ("k_out", k_out)):
            _heads(name, t, 3, dev)
            if t.dtype != q.dtype:
                _fail(f"{name} must be {q.dtype} as q is, got {t.dtype}")
        tokens, _, D = q.shape
        if k.size(0) != tokens or k.size(2) != D:
            _fail(f"k must be ({tokens}, heads, {D}) for q {tuple(q.shape)}, got "
                  f"{tuple(k.shape)}")
        if q_out.shape != q.shape or k_out.shape != k.shape:
            _fail(f"the outputs must have the inputs' shapes {tuple(q.shape)} and "
                  f"{tuple(k.shape)}, got {tuple(q_out.shape)} and {tuple(k_out.shape)}")
        wdt = None
        for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
            if w is None:
                continue
            _gpu(name, w, dev)
            if tuple(w.shape) != (D,) or not w.is_contiguous():
                _fail(f"{name} must be contiguous of shape ({D},), got {tuple(w.shape)}")
            if w.dtype not in _DTYPES or (wdt is not None and w.dtype != wdt):
                _fail("the weights must share a type, float16, bfloat16 or float32, got "
                      f"{w.dtype}")
            wdt = w.dtype
        a = _capi.CqNormRope()
        if cos is not None or sin is not None or positions is not None:
            if cos is None or sin is None or positions is None:
                _fail("cos, sin and positions come together")
            for name, t in (("cos", cos), ("sin", sin)):
                _gpu(name, t, dev)
                if t.dtype != torch.float32 or t.dim() != 2 or not t.is_contiguous():
                    _fail(f"{name} must be a contiguous float32 table (rows, R/2), got "
                          f"{t.dtype} {tuple(t.shape)}")
            if cos.shape != sin.shape or cos.size(0) < 1:
                _fail(f"cos and sin must have one shape, got {tuple(cos.shape)} and "
                      f"{tuple(sin.shape)}")
            if not 2 <= 2 * cos.size(1) <= D:
                _fail(f"the tables turn {2 * cos.size(1)} dims, of heads of {D}")
            _gpu("positions", positions, dev)
            if positions.dtype not in (torch.int32, torch.int64) \
                    or tuple(positions.shape) != (tokens,) or not positions.is_contiguous():
                _fail(f"positions must be contiguous int32 or int64 ({tokens},), got "
                      f"{positions.dtype} {tuple(positions.shape)}")
            a.cos_table, a.sin_table = cos.data_ptr(), sin.data_ptr()
            a.positions = positions.data_ptr()
            a.table_rows, a.rot_dim = cos.size(0), 2 * cos.size(1)
            a.positions_64 = positions.dtype == torch.int64
        elif wdt is None:
            _fail("nothing to do: neither weights nor tables")
        if tokens == 0:
            return
        a.q, a.k, a.q_out, a.k_out = (t.data_ptr() for t in (q, k, q_out, k_out))
        a.q_token_stride, a.q_head_stride = q.stride(0), q.stride(1)
        a.k_token_stride, a.k_head_stride = k.stride(0), k.stride(1)
        a.q_out_token_stride, a.q_out_head_stride = q_out.stride(0), q_out.stride(1)
        a.k_out_token_stride, a.k_out_head_stride = k_out.stride(0), k_out.stride(1)
        a.q_weight = None if q_weight is None else q_weight.data_ptr()
        a.k_weight = None if k_weight is None else k_weight.data_ptr()
        a.tokens, a.q_heads, a.k_heads, a.head_dim = tokens, q.size(1), k.size(1), D
        a.dtype = _DTYPES[q.dtype]
        a.weight_dtype = _DTYPES[wdt or torch.float32]
        a.interleaved, a.eps = interleaved, eps
        _check(_on_device(dev, lambda s: self._lib.cq_qk_norm_rope(ctypes.byref(a), s)),
               "qk_norm_rope")

    # ---- the cache ----
    def _slots(self, cache, block_table, starts, counts, batch: int, tokens: int):
        if not isinstance(cache, KVCache):
            _fail(f"cache must be a KVCache, got {type(cache).__name__}")
        dev = cache.device
        _table("block_table", block_table, batch, dev)
        _ints("starts", starts, (batch,), dev)
        if counts is not None:
            _ints("counts", counts, (batch,), dev)
        return _capi.CqKvSlots(
            block_table.data_ptr(), starts.data_ptr(),
            None if counts is None else counts.data_ptr(), block_table.stride(0),
            block_table.size(1), batch, tokens)

    def append(self, cache: KVCache, k: torch.Tensor, v: torch.Tensor,
               block_table: torch.Tensor, starts: torch.Tensor,
               counts: Optional[torch.Tensor] = None) -> None:
        """Quantizes k and v (batch, tokens, heads, D) into the cache: token t
        of sequence b goes to position starts[b] + t, for t < counts[b] (all
        tokens if None).  block_table int32 (batch, pages), starts and counts
        int32 (batch,).  A token whose position or page is out of range is not
        written; pages written belong to one sequence each."""
        if not isinstance(cache, KVCache):
            _fail(f"cache must be a KVCache, got {type(cache).__name__}")
        if self._fast is not None and cache.fast is not None \
                and self._fast.append(cache.fast, k, v, block_table, starts, counts):
            return
        for name, t in (("k", k), ("v", v)):
            _heads(name, t, 4, cache.device)
            if t.dtype != k.dtype or t.shape != k.shape:
                _fail(f"k and v must share type and shape, got {k.dtype} {tuple(k.shape)} "
                      f"and {t.dtype} {tuple(t.shape)}")
        if k.size(2) != cache.heads or k.size(3) != cache.head_dim:
            _fail(f"k and v must be (batch, tokens, {cache.heads}, {cache.head_dim}), got "
                  f"{tuple(k.shape)}")
        batch, tokens = k.size(0), k.size(1)
        slots = self._slots(cache, block_table, starts, counts, batch, tokens)
        if batch == 0 or tokens == 0:
            return
        ks, vs = k.stride(), v.stride()
        _check(_on_device(cache.device, lambda s: self._lib.cq_kv_append(
            ctypes.byref(cache.c), ctypes.byref(slots), _DTYPES[k.dtype], k.data_ptr(),
            ks[0], ks[1], ks[2], v.data_ptr(), vs[0], vs[1], vs[2], s)), "append")

    def read(self, cache: KVCache, block_table: torch.Tensor, starts: torch.Tensor,
             counts: Optional[torch.Tensor], tokens: int,
             dtype: torch.dtype = torch.float16) -> tuple[torch.Tensor, torch.Tensor]:
        """The cached values of tokens starts[b] .. starts[b] + counts[b] of
        each sequence as (k, v), each (batch, tokens, heads, D) of `dtype`;
        zeros past the count and where no page is."""
        if not isinstance(cache, KVCache):
            _fail(f"cache must be a KVCache, got {type(cache).__name__}")
        if self._fast is not None and cache.fast is not None:
            got = self._fast.read(cache.fast, block_table, starts, counts, tokens, dtype)
            if got is not None:
                return got
        if dtype not in _DTYPES:
            _fail(f"dtype must be float16, bfloat16 or float32, got {dtype}")
        if isinstance(tokens, bool) or not isinstance(tokens, int) \
                or not 0 <= tokens < 2 ** 31:
            _fail(f"tokens must be an int in [0, 2^31), got {tokens!r}")
        batch = starts.size(0) if isinstance(starts, torch.Tensor) and starts.dim() else 0
        slots = self._slots(cache, block_table, starts, counts, batch, tokens)
        shape = (batch, tokens, cache.heads, cache.head_dim)
        k = torch.empty(shape, dtype=dtype, device=cache.device)
        v = torch.empty(shape, dtype=dtype, device=cache.device)
        if k.numel():
            _check(_on_device(cache.device, lambda s: self._lib.cq_kv_read(
                ctypes.byref(cache.c), ctypes.byref(slots), _DTYPES[dtype], k.data_ptr(),
                v.data_ptr(), s)), "read")
        return k, v

    # ---- packed batches ----
    def place(self, block_table: torch.Tensor, starts: torch.Tensor, counts: torch.Tensor,
              tokens: int, page_size: int, free_pages: torch.Tensor,
              taken: Optional[torch.Tensor] = None, *,
              held: Optional[torch.Tensor] = None) -> Placed | PlacedHeld:
        """Pages, positions and slots for a packed batch of `tokens` rows in
        which sequence b adds counts[b] tokens to the starts[b] that it has.

        Sequence b holds the first ceil(starts[b] / page_size) entries of its
        row of block_table int32 (batch, pages); the pages that it needs beyond
        come from free_pages int32 (n,), in the sequences' order, from entry
        taken[0] (int32 (1,), 0 if None) on, and are written into the table (-1
        where the list has ended).  The result's `taken` says how many entries
        are gone then: above n the list did not suffice.  It may be the next
        call's `taken`.  A token without a page, or past the table, has slot -1,
        and so have rows behind the last sequence.  Tokens that do not fit
        `tokens` rows are not placed, and `lengths` does not count them.
        Negative starts and counts are zero.

        `held` int32 (batch,) says how many entries of its row a sequence owns
        where those may be more than its start needs, as when drafted tokens were
        given up: these entries are used before pages are taken from the list (without
        it they are overwritten and their pages lost to the list).  The result is
        then a PlacedHeld, whose `held` is the next call's, as its `taken` is; a
        sequence whose pages go back to the list starts with 0."""
        if self._step is not None:
            got = self._step.place(block_table, starts, counts, tokens, page_size, free_pages,
                                   taken, held)
            if got is not None:
                return Placed(*got) if held is None else PlacedHeld(*got)
        if not isinstance(block_table, torch.Tensor):
            _fail(f"block_table must be a tensor, got {type(block_table).__name__}")
        dev = block_table.device
        batch = block_table.size(0) if block_table.dim() == 2 else 0
        _table("block_table", block_table, batch, dev)
        _ints("starts", starts, (batch,), dev)
        _ints("counts", counts, (batch,), dev)
        _count("tokens", tokens)
        if isinstance(page_size, bool) or not hasattr(page_size, "__index__") \
                or page_size not in PAGE_SIZES:
            _fail(f"the page size must be one of {PAGE_SIZES}, got {page_size!r}")
        _gpu("free_pages", free_pages, dev)
        _ints("free_pages", free_pages, (free_pages.numel(),), dev)
        if taken is not None:
            _ints("taken", taken, (1,), dev)
        if held is not None:
            _ints("held", held, (batch,), dev)

        def ints(n, dtype=torch.int32):
            return torch.empty(n, dtype=dtype, device=dev)

        p = Placed(ints(tokens, torch.int64), ints(tokens), ints(batch + 1), ints(batch),
                   ints(1))
        if held is not None:
            p = PlacedHeld(*p, ints(batch))
        if batch == 0:
            p.slots.fill_(-1)
            p.positions.zero_()
            p.offsets.zero_()
            p.taken.zero_()
            return p if taken is None else p._replace(taken=taken.clamp(min=0))
        a = _capi.CqPlace(
            starts.data_ptr(), counts.data_ptr(), free_pages.data_ptr() or None,
            None if taken is None else taken.data_ptr(), block_table.data_ptr(),
            p.slots.data_ptr() or None, p.positions.data_ptr() or None, p.offsets.data_ptr(),
            p.lengths.data_ptr(), p.taken.data_ptr(), block_table.stride(0), tokens,
            free_pages.numel(), block_table.size(1), batch, page_size)
        _check(_on_device(dev, lambda s: self._lib.cq_place_held(
            ctypes.byref(a), None if held is None else held.data_ptr(),
            None if held is None else p.held.data_ptr(), s)), "place")
        return p

    def append_rows(self, cache: KVCache, k: torch.Tensor, v: torch.Tensor,
                    slots: torch.Tensor) -> None:
        """Quantizes packed k and v (tokens, heads, D) into the cache: row t
        goes to slots[t] = page * page_size + offset (int64 (tokens,)), as `place`
        gives them.  A row with a slot outside the cache (-1) is not written; no
        two rows have one slot.  Accepted drafts are closed up this way: their
        rows again, to the slots behind one another, the others' -1."""
        if not isinstance(cache, KVCache):
            _fail(f"cache must be a KVCache, got {type(cache).__name__}")
        if self._step is not None and cache.fast is not None \
                and self._step.append_rows(cache.fast, k, v, slots):
            return
        for name, t in (("k", k), ("v", v)):
            _heads(name, t, 3, cache.device)
            if t.dtype != k.dtype or t.shape != k.shape:
                _fail(f"k and v must share type and shape, got {k.dtype} {tuple(k.shape)} "
                      f"and {t.dtype} {tuple(t.shape)}")
        tokens = k.size(0)
        if k.size(1) != cache.heads or k.size(2) != cache.head_dim:
            _fail(f"k and v must be (tokens, {cache.heads}, {cache.head_dim}), got "
                  f"{tuple(k.shape)}")
        _gpu("slots", slots, cache.device)
        if slots.dtype != torch.int64 or tuple(slots.shape) != (tokens,) \
                or not slots.is_contiguous():
            _fail(f"slots must be contiguous int64 ({tokens},), got {slots.dtype} "
                  f"{tuple(slots.shape)}")
        if tokens == 0:
            return
        ks, vs = k.stride(), v.stride()
        _check(_on_device(cache.device, lambda s: self._lib.cq_kv_append_rows(
            ctypes.byref(cache.c), _DTYPES[k.dtype], tokens, slots.data_ptr(), k.data_ptr(),
            ks[0], ks[1], v.data_ptr(), vs[0], vs[1], s)), "append_rows")

    def prompt(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
               offsets: torch.Tensor, *, k_offsets: Optional[torch.Tensor] = None,
               causal: bool = True, scale: Optional[float] = None) -> torch.Tensor:
        """Attention of packed sequences over keys and values that lie beside
        them, into a new tensor of q's shape and type.  See prompt_into."""
        return self._prompt(q, k, v, offsets, None, k_offsets, causal, scale)

    def prompt_into(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                    offsets: torch.Tensor, out: torch.Tensor, *,
                    k_offsets: Optional[torch.Tensor] = None, causal: bool = True,
                    scale: Optional[float] = None) -> None:
        """Attention of packed sequences into a given contiguous `out` that starts at
        16 bytes.

        q (tokens, Hq, D), k and v (keys, H, D), float16 or bfloat16, as they are
        before they enter a cache: nothing is quantized.  Sequence b's n queries
        are the rows offsets[b] .. offsets[b + 1] (int32 (batch + 1,), ascending
        from 0), its m keys the rows k_offsets[b] .. k_offsets[b + 1] of k and v
        (offsets, if None; with more keys than queries the earlier ones are of
        earlier chunks).  Query t sees the keys up to m - n + t, or all m without
        `causal`; query head h reads key head h // (Hq // H).  `scale` multiplies
        the scores (default D ** -0.5).  Scores, statistics and sums are FP32;
        each weight is rounded to the type before it multiplies v, the result
        once.  A key that a query does not see leaves no trace, whatever it
        holds.  Queries that see nothing and rows of no sequence give zeros."""
        if out is None:
            _fail("out must be a tensor, got NoneType")
        self._prompt(q, k, v, offsets, out, k_offsets, causal, scale)

    def _prompt(self, q, k, v, offsets, out, k_offsets, causal, scale):
        causal = bool(causal)
        if scale is not None:
            scale = _number("scale", scale)
        if self._step is not None:
            got = self._step.prompt(q, k, v, offsets, out, k_offsets, causal, scale)
            if got is not None:
                return got
        if not isinstance(q, torch.Tensor):
            _fail(f"q must be a tensor, got {type(q).__name__}")
        dev = q.device
        for name, t in (("q", q), ("k", k), ("v", v)):
            _heads(name, t, 3, dev)
            if t.dtype != q.dtype or t.dtype == torch.float32:
                _fail(f"q, k and v must share float16 or bfloat16, got {q.dtype} and {t.dtype}")
        tokens, hq, D = q.shape
        keys, heads = k.size(0), k.size(1)
        if v.shape != k.shape or k.size(2) != D:
            _fail(f"k and v must be (keys, heads, {D}), got {tuple(k.shape)} and "
                  f"{tuple(v.shape)}")
        if D not in HEAD_DIMS:
            _fail(f"the head size must be one of {HEAD_DIMS}, got {D}")
        if heads < 1 or hq < 1 or hq % heads:
            _fail(f"q's heads must be a multiple of k's, got {hq} and {heads}")
        _gpu("offsets", offsets, dev)
        if offsets.dim() != 1 or offsets.numel() < 1:
            _fail(f"offsets must be (batch + 1,), got {tuple(offsets.shape)}")
        batch = offsets.numel() - 1
        _ints("offsets", offsets, (batch + 1,), dev)
        if k_offsets is not None:
            _ints("k_offsets", k_offsets, (batch + 1,), dev)
        elif keys != tokens:
            _fail(f"without k_offsets k and v have q's {tokens} rows, got {keys}")
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        _gpu("out", out, dev)
        if out.dtype != q.dtype or out.shape != q.shape or not out.is_contiguous():
            _fail(f"out must be contiguous {q.dtype} {tuple(q.shape)}, got {out.dtype} "
                  f"{tuple(out.shape)}")
        if tokens == 0:
            return out
        if batch == 0:
            return out.zero_()

        def aligned(t, most):
            # the kernels read 16 bytes of a head at once (and the strides of no keys
            # are checked like any others')
            if not (t.data_ptr() % 16 or any(s % 8 for s in t.stride()[:2])
                    or t.stride(0) > most):
                return t
            return torch.empty(t.shape, dtype=t.dtype, device=dev).copy_(t)

        q, k, v = aligned(q, 2 ** 40), aligned(k, 2 ** 24), aligned(v, 2 ** 24)
        a = _capi.CqPrompt(
            q.data_ptr(), k.data_ptr() or None, v.data_ptr() or None, out.data_ptr(),
            q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1),
            offsets.data_ptr(), None if k_offsets is None else k_offsets.data_ptr(), tokens,
            keys, batch, hq, heads, D, _DTYPES[q.dtype], causal,
            D ** -0.5 if scale is None else scale)
        _check(_on_device(dev, lambda s: self._lib.cq_prompt_attention(ctypes.byref(a), s)),
               "prompt")
        return out

    # ---- attention ----
    def forward(self, q: torch.Tensor, cache: KVCache, block_table: torch.Tensor,
                lengths: torch.Tensor, counts: Optional[torch.Tensor] = None, *,
                prefix: Optional[tuple[torch.Tensor, int]] = None,
                scale: Optional[float] = None,
                tree: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of q (batch, tokens, Hq, D), float16 or bfloat16, over the
        cache, into a new tensor of q's shape and type.  See forward_into."""
        if scale is not None:
            scale = _number("scale", scale)
        got = self._fast_forward(q, cache, block_table, lengths, None, counts, prefix, scale,
                                 tree)
        if got is not None:
            return got
        if not isinstance(q, torch.Tensor):
            _fail(f"q must be a tensor, got {type(q).__name__}")
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        self._forward(q, cache, block_table, lengths, out, counts, prefix, scale, tree)
        return out

    def forward_into(self, q: torch.Tensor, cache: KVCache, block_table: torch.Tensor,
                     lengths: torch.Tensor, out: torch.Tensor,
                     counts: Optional[torch.Tensor] = None, *,
                     prefix: Optional[tuple[torch.Tensor, int]] = None,
                     scale: Optional[float] = None,
                     tree: Optional[torch.Tensor] = None) -> None:
        """Attention into a given contiguous `out` that starts at 16 bytes.

        Sequence b holds lengths[b] tokens in the pages block_table[b]; the
        last counts[b] of them (all `tokens` if None) are the call's own: query
        t sits at position lengths[b] - counts[b] + t and sees the positions up
        to it.  Query head h reads cache head h // (Hq // heads).  `prefix`
        (pages int32 (n,), length) names tokens that every query of every
        sequence sees before its own: they are read once for the whole batch,
        and `lengths` does not count them.  `scale` multiplies the scores
        (default D ** -0.5).

        `tree` int64 (batch, tokens, ceil(tokens / 64)) says which of the call's
        tokens each of them sees, in the place of those up to itself: query t sees
        token j if bit j % 64 of tree[b, t, j // 64] is set (a drafted token's own
        bit and its ancestors'), and everything ahead of the call's tokens.

        Scores, statistics and sums are FP32, from q held
        in FP16 times a power of two of its row; each probability times its V
        scale is rounded to FP16 before it multiplies V's codes, the result once
        to q's type.  A query that sees nothing, or lies past counts[b], gives
        zeros, whatever it holds."""
        if scale is not None:
            scale = _number("scale", scale)
        if out is not None and self._fast_forward(q, cache, block_table, lengths, out, counts,
                                                  prefix, scale, tree) is not None:
            return
        self._forward(q, cache, block_table, lengths, out, counts, prefix, scale, tree)

    def _fast_forward(self, q, cache, block_table, lengths, out, counts, prefix, scale, tree):
        if self._fast is None or not isinstance(cache, KVCache) or cache.fast is None:
            return None
        pages, n = None, 0
        if prefix is not None:
            pages, n = _pair(prefix)
            if type(n) is not int or not 0 <= n < 2 ** 31 or pages is None:
                return None
        if scale is None:
            scale = cache.head_dim ** -0.5
        return self._fast.forward(cache.fast, q, block_table, lengths, counts, out, pages, n,
                                  scale, tree)

    def _forward(self, q, cache, block_table, lengths, out, counts, prefix, scale, tree) -> None:
        if not isinstance(cache, KVCache):
            _fail(f"cache must be a KVCache, got {type(cache).__name__}")
        dev = cache.device
        _heads("q", q, 4, dev)
        if q.dtype not in (torch.float16, torch.bfloat16):
            _fail(f"q must be float16 or bfloat16, got {q.dtype}")
        batch, tokens, hq, D = q.shape
        if D != cache.head_dim or hq < 1 or hq % cache.heads:
            _fail(f"q must be (batch, tokens, a multiple of {cache.heads}, "
                  f"{cache.head_dim}), got {tuple(q.shape)}")
        _gpu("out", out, dev)
        if out.dtype != q.dtype or out.shape != q.shape or not out.is_contiguous():
            _fail(f"out must be contiguous {q.dtype} {tuple(q.shape)}, got {out.dtype} "
                  f"{tuple(out.shape)}")
        _table("block_table", block_table, batch, dev)
        _ints("lengths", lengths, (batch,), dev)
        if counts is not None:
            _ints("counts", counts, (batch,), dev)
        if tree is not None:
            _gpu("tree", tree, dev)
            shape = (batch, tokens, (tokens + 63) // 64)
            if tree.dtype != torch.int64 or tuple(tree.shape) != shape \
                    or not tree.is_contiguous():
                _fail(f"tree must be contiguous int64 {shape}, got {tree.dtype} "
                      f"{tuple(tree.shape)}")
        a = _capi.CqAttention()
        if prefix is not None:
            pages, n = _pair(prefix)
            _gpu("the prefix's pages", pages, dev)
            if pages.dtype != torch.int32 or pages.dim() != 1 or not pages.is_contiguous():
                _fail(f"the prefix's pages must be contiguous int32 (n,), got {pages.dtype} "
                      f"{tuple(pages.shape)}")
            if isinstance(n, bool) or not isinstance(n, int) \
                    or not 0 <= n <= min(pages.numel() * cache.page_size, 2 ** 31 - 1):
                _fail(f"the prefix's length must be an int within its {pages.numel()} "
                      f"pages, got {n!r}")
            a.prefix_table = pages.data_ptr() if n else None
            a.prefix_cols, a.prefix_len = pages.numel(), n
        if batch == 0 or tokens == 0:
            return
        if q.data_ptr() % 16 or any(s % 8 for s in q.stride()[:3]):
            # the kernels read 16 bytes of a head at once; a q that is contiguous
            # may still start, or have a dimension of one, off them
            q = torch.empty(q.shape, dtype=q.dtype, device=dev).copy_(q)
        a.q, a.out = q.data_ptr(), out.data_ptr()
        a.q_batch_stride, a.q_token_stride, a.q_head_stride = q.stride()[:3]
        a.table, a.lengths = block_table.data_ptr(), lengths.data_ptr()
        a.counts = None if counts is None else counts.data_ptr()
        a.table_stride, a.table_cols = block_table.stride(0), block_table.size(1)
        a.batch, a.tokens, a.q_heads, a.dtype = batch, tokens, hq, _DTYPES[q.dtype]
        a.softmax_scale = D ** -0.5 if scale is None else scale
        sizes = (self._lib.cq_attention_workspace if tree is None
                 else self._lib.cq_attention_tree_workspace)
        need = sizes(ctypes.byref(cache.c), ctypes.byref(a))
        if need < 0:
            _check(-need, "forward")
        ws = None
        if need:
            ws = torch.empty(need, dtype=torch.uint8, device=dev)
            a.workspace, a.workspace_bytes = ws.data_ptr(), need
        if tree is None:
            _check(_on_device(dev, lambda s: self._lib.cq_attention(
                ctypes.byref(cache.c), ctypes.byref(a), s)), "forward")
        else:
            _check(_on_device(dev, lambda s: self._lib.cq_attention_tree(
                ctypes.byref(cache.c), ctypes.byref(a), tree.data_ptr(), s)), "forward")


_ATTENTION: Optional[AttentionExt] = None


def get_attention() -> AttentionExt:
    """The process's AttentionExt (`build("attention")`)."""
    global _ATTENTION
    if _ATTENTION is None:
        _ATTENTION = AttentionExt()
    return _ATTENTION
