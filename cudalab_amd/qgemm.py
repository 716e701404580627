"""INT8 products of many tokens, over the C ABI: `build("qgemm")` returns the one
`QgemmExt`.  No counterpart in the reference, whose products take one vector.

    gemm = build("qgemm")
    codes, scales = gemm.quantize_tokens(x)              # once for q, k and v
    y = gemm.forward(codes, scales, W_q, scale)          # (tokens, N)

W_q int8 (N, K) and scale float32 (N,) are what `qgemv_quantize.quantize_w` gives
and the INT8 GEMV takes: a model keeps one copy for prompts and single tokens.
Unlike there the activations are quantized too, with a scale for each token.

Checks run on the host before anything is launched and raise RuntimeError.
Launches go on the current torch stream of W_q's (x's) device, work inside a HIP
graph, and keep nothing between calls.  Each call is first offered to the fast
path (csrc/cq_pystep.h), as the other operators' are.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _capi
from .attention import _DTYPES, _check, _fail, _gpu
from .ext import _on_device, fast_module_or_none

# sums of more products of two codes would not fit 32 bits
MAX_K = 131071


class QgemmExt:
    """Quantized tokens, and their products with INT8 weights."""

    def __init__(self) -> None:
        self._lib = _capi.load()
        mod = fast_module_or_none()
        self._fast = mod and mod.QgemmCalls(*(_capi.entry_address(n) for n in (
            "cq_quantize_tokens", "cq_qgemm", "cq_qgemm_workspace", "cq_last_error")))

    def quantize_tokens(self, x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """(codes int8 (tokens, K), scales float32 (tokens,)) of x (tokens, K),
        float16, bfloat16 or float32, the last dimension contiguous.  Per token,
        every operation rounded to FP32:
            scale = amax * fl(1 / 127), code = round_half_even(x * fl(1 / scale))
        A token whose amax is below 2^-100 gets scale 0 and codes 0; one with NaN
        or Inf gets scale NaN, and its row of every product becomes NaN."""
        if self._fast is not None:
            got = self._fast.quantize(x)
            if got is not None:
                return got
        if not isinstance(x, torch.Tensor):
            _fail(f"x must be a tensor, got {type(x).__name__}")
        _gpu("x", x, x.device)
        if x.dim() != 2 or x.dtype not in _DTYPES:
            _fail(f"x must be (tokens, K) of float16, bfloat16 or float32, got {x.dtype} "
                  f"{tuple(x.shape)}")
        tokens, K = x.shape
        if K < 1:
            _fail("K must be > 0, got 0")
        if K > 1 and x.stride(1) != 1:
            _fail("the last dimension of x must be contiguous")
        codes = torch.empty(tokens, K, dtype=torch.int8, device=x.device)
        scales = torch.empty(tokens, dtype=torch.float32, device=x.device)
        if tokens:
            _check(_on_device(x.device, lambda s: self._lib.cq_quantize_tokens(
                _DTYPES[x.dtype], x.data_ptr(), x.stride(0), tokens, K, codes.data_ptr(),
                scales.data_ptr(), s)), "quantize_tokens")
        return codes, scales

    def forward(self, codes: torch.Tensor, scales: torch.Tensor, W_q: torch.Tensor,
                scale: torch.Tensor, dtype: torch.dtype = torch.float16) -> torch.Tensor:
        """The product into a new tensor (tokens, N) of `dtype`.  See forward_into."""
        if self._fast is not None:
            got = self._fast.forward(codes, scales, W_q, scale, None, dtype)
            if got is not None:
                return got
        if dtype not in _DTYPES:
            _fail(f"dtype must be float16, bfloat16 or float32, got {dtype}")
        if not isinstance(W_q, torch.Tensor) or not isinstance(codes, torch.Tensor):
            _fail("codes and W_q must be tensors")
        _gpu("W_q", W_q, W_q.device)
        if codes.dim() != 2 or W_q.dim() != 2:
            _fail(f"codes and W_q must be 2-D, got {codes.dim()}-D and {W_q.dim()}-D")
        out = torch.empty(codes.size(0), W_q.size(0), dtype=dtype, device=W_q.device)
        self._forward(codes, scales, W_q, scale, out)
        return out

    def forward_into(self, codes: torch.Tensor, scales: torch.Tensor, W_q: torch.Tensor,
                     scale: torch.Tensor, out: torch.Tensor) -> None:
        """The product into a given contiguous `out` (tokens, N), float16, bfloat16
        or float32, that starts at 16 bytes:

            out[t, n] = (sum_k codes[t, k] W_q[n, k]) * scales[t] * scale[n]

        codes int8 (tokens, K), rows any distance apart, and scales float32
        (tokens,) as quantize_tokens gives them; W_q int8 (N, K) and scale float32
        (N,) contiguous.  The sum is a whole number (K at most 131071), the
        products are FP32, rounded once to out's type, so a result depends on
        nothing but its row and its channel."""
        if self._fast is not None and out is not None \
                and self._fast.forward(codes, scales, W_q, scale, out, None) is not None:
            return
        self._forward(codes, scales, W_q, scale, out)

    def _forward(self, codes, scales, W_q, scale, out) -> None:
        if not isinstance(W_q, torch.Tensor):
            _fail(f"W_q must be a tensor, got {type(W_q).__name__}")
        dev = W_q.device
        for name, t in (("W_q", W_q), ("codes", codes), ("scale", scale), ("scales", scales),
                        ("out", out)):
            _gpu(name, t, dev)
        for name, t in (("W_q", W_q), ("codes", codes)):
            if t.dim() != 2 or t.dtype != torch.int8:
                _fail(f"{name} must be 2-D int8, got {t.dtype} {tuple(t.shape)}")
        N, K = W_q.shape
        tokens = codes.size(0)
        if N < 1 or K < 1 or K > MAX_K:
            _fail(f"W_q must be (N, K) with N > 0 and 0 < K <= {MAX_K}, got {tuple(W_q.shape)}")
        if not W_q.is_contiguous():
            _fail("W_q must be contiguous")
        if codes.size(1) != K:
            _fail(f"codes must be (tokens, {K}), got {tuple(codes.shape)}")
        if K > 1 and codes.stride(1) != 1 or tokens > 1 and codes.stride(0) < K:
            _fail("the rows of codes must be contiguous and apart")
        for name, t, n in (("scale", scale, N), ("scales", scales, tokens)):
            if t.dtype != torch.float32 or tuple(t.shape) != (n,) or not t.is_contiguous():
                _fail(f"{name} must be contiguous float32 ({n},), got {t.dtype} "
                      f"{tuple(t.shape)}")
        if out.dtype not in _DTYPES or tuple(out.shape) != (tokens, N) \
                or not out.is_contiguous():
            _fail(f"out must be contiguous float16, bfloat16 or float32 ({tokens}, {N}), got "
                  f"{out.dtype} {tuple(out.shape)}")
        if tokens == 0:
            return
        a = _capi.CqQgemm(
            codes.data_ptr(), scales.data_ptr(), W_q.data_ptr(), scale.data_ptr(),
            out.data_ptr(), max(codes.stride(0), K), tokens, N, K, None, 0, _DTYPES[out.dtype])
        need = self._lib.cq_qgemm_workspace(ctypes.byref(a))
        if need < 0:
            _check(-need, "forward")
        ws = None
        if need:
            ws = torch.empty(need, dtype=torch.uint8, device=dev)
            a.workspace, a.workspace_bytes = ws.data_ptr(), need
        _check(_on_device(dev, lambda s: self._lib.cq_qgemm(ctypes.byref(a), s)), "forward")


_QGEMM: Optional[QgemmExt] = None


def get_qgemm() -> QgemmExt:
    """The process's QgemmExt (`build("qgemm")`)."""
    global _QGEMM
    if _QGEMM is None:
        _QGEMM = QgemmExt()
    return _QGEMM
