"""GPU tests of the INT8 products of many tokens: codes, scales and results bit
for bit against the definition (whole sums, FP32 products, one rounding)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from attention_oracle import quantize
from conftest import announce

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def gemm(cuda):
    from cudalab_amd.build import build
    return build("qgemm")


def _want(codes, scales, w, scale, dtype):
    """On the CPU: sums in int64 (FP64 holds them exactly), then FP32."""
    s = codes.cpu().double() @ w.cpu().double().T
    with np.errstate(all="ignore"):
        y = s.float() * scales.cpu()[:, None] * scale.cpu()[None]
    return y.to(dtype)


def _same(got, want, what=""):
    got = got.cpu()
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan), what
    assert torch.equal(got[~nan], want[~nan]), (
        what, int((got != want).sum()), np.argwhere((got != want).numpy())[:3].tolist())


def _operands(m, n, k, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int8),
            torch.rand(m, generator=g) * 0.02 + 1e-4,
            torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8),
            torch.rand(n, generator=g) * 0.01 + 1e-4)


def _check(gemm, m, n, k, dtype="fp16", seed=0):
    announce(f"qgemm m={m} n={n} k={k} {dtype}")
    ops = _operands(m, n, k, seed)
    got = gemm.forward(*(t.cuda() for t in ops), DT[dtype])
    _same(got, _want(*ops, DT[dtype]), f"{m} {n} {k}")


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 48, 49, 64, 65, 128, 129, 200, 300])
@pytest.mark.parametrize("n,k", [(1, 1), (3, 16), (64, 128), (130, 144), (257, 640), (33, 1000)])
def test_sizes(gemm, dtype, m, n, k):
    _check(gemm, m, n, k, dtype)


@pytest.mark.parametrize("k", [2, 3, 5, 15, 17, 31, 63, 65, 100, 127, 129, 130, 255, 257, 1026, 4100])
@pytest.mark.parametrize("m,n", [(5, 70), (70, 67), (140, 260)])
def test_every_kind_of_row(gemm, m, n, k):
    """Rows that start at words, at bytes, and end anywhere."""
    _check(gemm, m, n, k)


@pytest.mark.parametrize("m,n,k", [(700, 4100, 256), (1500, 8200, 260), (257, 12345, 131),
                                   (2050, 6161, 128), (35, 8192, 2048), (64, 1024, 8192),
                                   (1, 28672, 512), (130, 512, 8192), (513, 1024, 4096)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_large(gemm, m, n, k, dtype):
    _check(gemm, m, n, k, dtype)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("m,n,k", [(120, 8000, 256), (250, 8100, 516), (500, 8190, 132),
                                   (777, 5003, 1028), (500, 11008, 260), (1500, 5001, 388),
                                   (1300, 8201, 320), (2000, 9000, 4)])
def test_every_tile(gemm, m, n, k, dtype):
    """Sizes that take each of the tiles, with edges in both directions."""
    _check(gemm, m, n, k, dtype)


def test_longest_rows(gemm):
    """The largest sums that 32 bits hold, and one more k is refused."""
    k = 131071
    for m in (3, 150):
        x = torch.full((m, k), -128, dtype=torch.int8)
        w = torch.full((5, k), -128, dtype=torch.int8)
        w[1] = 127
        w[2, ::2] = 127
        xs, ws = torch.ones(m), torch.ones(5)
        announce(f"qgemm longest rows m={m}")
        _same(gemm.forward(x.cuda(), xs.cuda(), w.cuda(), ws.cuda(), torch.float32),
              _want(x, xs, w, ws, torch.float32))
    x, w = (torch.zeros(2, k + 1, dtype=torch.int8, device="cuda") for _ in range(2))
    with pytest.raises(RuntimeError):
        gemm.forward(x, torch.ones(2, device="cuda"), w, torch.ones(2, device="cuda"))


@pytest.mark.parametrize("k,stride", [(100, 100), (100, 112), (96, 101), (128, 4096),
                                      (64, 2 ** 22 + 8)])
def test_rows_of_codes_apart(gemm, k, stride):
    """Rows of codes any distance apart and at any byte; what lies between is
    not read into a result."""
    for m in (7, 140):
        if m * stride > 2 ** 28:
            continue
        x, xs, w, ws = _operands(m, 70, k)
        for off in (0, 1, 4, 16):
            wide = torch.full((m * stride + off + k,), 127, dtype=torch.int8, device="cuda")
            dev = wide[off:].as_strided((m, k), (stride, 1))
            dev.copy_(x)
            announce(f"qgemm rows apart m={m} k={k} stride={stride} off={off}")
            _same(gemm.forward(dev, xs.cuda(), w.cuda(), ws.cuda()),
                  _want(x, xs, w, ws, torch.float16))


def test_nothing_else_is_written(gemm):
    """Outputs inside a larger buffer, weights at odd bytes."""
    for m, n, k in ((3, 5, 33), (40, 100, 64), (130, 131, 100)):
        x, xs, w, ws = _operands(m, n, k)
        big = torch.full((m * n + 64,), 7.0, dtype=torch.float16, device="cuda")
        out = big[8:8 + m * n].view(m, n)
        raw = torch.zeros(n * k + 16, dtype=torch.int8, device="cuda")
        wd = raw[3:3 + n * k].view(n, k)
        wd.copy_(w)
        announce(f"qgemm into a buffer {m} {n} {k}")
        gemm.forward_into(x.cuda(), xs.cuda(), wd, ws.cuda(), out)
        _same(out, _want(x, xs, w, ws, torch.float16))
        assert bool((big[:8] == 7).all()) and bool((big[8 + m * n:] == 7).all())


def test_special_scales(gemm):
    """NaN, Inf, zero and tiny scales are their row's or channel's alone; results
    past the type become Inf."""
    for m, n in ((9, 40), (140, 140)):
        x, xs, w, ws = _operands(m, n, 256)
        xs[1], xs[2], xs[3], xs[4] = float("nan"), float("inf"), 0.0, 1e30
        ws[5], ws[6], ws[7] = float("nan"), 0.0, 2.0 ** -120
        announce(f"qgemm special scales {m}")
        for dt in DT.values():
            _same(gemm.forward(x.cuda(), xs.cuda(), w.cuda(), ws.cuda(), dt),
                  _want(x, xs, w, ws, dt))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("k", [1, 7, 8, 100, 1000, 2048, 2049, 4096, 5000, 8192, 12345, 16384,
                               20000, 40001])
def test_quantize_tokens(gemm, dtype, k):
    g = torch.Generator().manual_seed(k)
    x = torch.randn(9, k, generator=g) * 10.0 ** torch.randint(-3, 3, (9, 1), generator=g)
    x[2] = 0
    x[3] = 2.0 ** -101
    x[4, k // 2] = float("nan")
    x[5, k - 1] = float("-inf")
    x[6] = torch.arange(k) % 255 - 127.0
    x[7, 0] = 3.0e38
    x = x.to(DT[dtype])
    announce(f"quantize_tokens {dtype} k={k}")
    codes, scales = gemm.quantize_tokens(x.cuda())
    want, scale = quantize(x.float().numpy(), 8)
    assert np.array_equal(codes.cpu().numpy().astype(np.int32), want)
    assert np.array_equal(scales.cpu().numpy(), scale, equal_nan=True)
    # rows apart, one element off 16 bytes
    wide = torch.full((9, k + 5), float("nan"), dtype=x.dtype, device="cuda")
    wide[:, 1:k + 1] = x.cuda()
    codes2, scales2 = gemm.quantize_tokens(wide[:, 1:k + 1])
    assert torch.equal(codes, codes2)
    assert torch.equal(scales.view(torch.int32), scales2.view(torch.int32))


def test_together_with_the_gemv_weights(gemm):
    """The weights that the INT8 GEMV takes, tokens quantized on the device: near
    the product of what was quantized."""
    from cudalab_amd.qgemv_quantize import quantize_w
    g = torch.Generator().manual_seed(1)
    W = (torch.randn(300, 512, generator=g) / 512 ** 0.5).half().cuda()
    x = torch.randn(50, 512, generator=g).half().cuda()
    wq, s = quantize_w(W)
    codes, scales = gemm.quantize_tokens(x)
    y = gemm.forward(codes, scales, wq, s)
    _same(y, _want(codes, scales, wq, s, torch.float16))
    # each operand is off by at most half a step of its row's
    exact = x.double().cpu() @ W.double().cpu().T
    bound = (x.double().cpu().abs() @ (s.cpu().double()[:, None] * 0.51).expand(-1, 512).T
             + (scales.cpu().double()[:, None] * 0.51).expand(-1, 512)
             @ (W.double().cpu().abs() + s.cpu().double()[:, None]).T)
    err = (y.double().cpu() - exact).abs()
    assert bool((err <= bound + exact.abs() * 2.0 ** -11).all())


def test_graph_streams_and_repeats(gemm):
    for m in (20, 200):
        x, xs, w, ws = (t.cuda() for t in _operands(m, 300, 512))
        h = torch.randn(m, 512, device="cuda").half()
        out = torch.empty(m, 300, dtype=torch.float16, device="cuda")

        def step():
            c, s = gemm.quantize_tokens(h)
            gemm.forward_into(c, s, w, ws, out)

        step()
        torch.cuda.synchronize()
        announce(f"qgemm in a graph m={m}")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        for i in range(3):
            h.copy_(torch.randn(m, 512, device="cuda"))
            g.replay()
            torch.cuda.synchronize()
            c, s = gemm.quantize_tokens(h)
            assert torch.equal(out, gemm.forward(c, s, w, ws))
        want = gemm.forward(x, xs, w, ws)
        torch.cuda.synchronize()
        side = [torch.cuda.Stream() for _ in range(2)]
        got = []
        for st in side:
            with torch.cuda.stream(st):
                got.append(gemm.forward(x, xs, w, ws))
        torch.cuda.synchronize()
        assert all(torch.equal(want, y) for y in got)


def test_empty_and_refusals(gemm):
    x, xs, w, ws = (t.cuda() for t in _operands(4, 6, 32))
    assert gemm.forward(x[:0], xs[:0], w, ws).shape == (0, 6)
    c, s = gemm.quantize_tokens(torch.zeros(0, 5, device="cuda").half())
    assert c.shape == (0, 5) and s.shape == (0,)
    good = dict(codes=x, scales=xs, W_q=w, scale=ws)
    for change in (dict(codes=None), dict(W_q=None), dict(codes=x.int()), dict(W_q=w.int()),
                   dict(codes=x[:, :31]), dict(codes=x[0]), dict(W_q=w[0]), dict(codes=x.cpu()),
                   dict(W_q=w.cpu()), dict(W_q=w.t()), dict(W_q=w[:, ::2], codes=x[:, ::2]),
                   dict(codes=x[:1].expand(4, 32)), dict(scales=xs[:3]), dict(scales=xs.half()),
                   dict(scale=ws[:5]), dict(scale=ws.double()), dict(scale=ws[None]),
                   dict(scales=None), dict(W_q=w[:0], scale=ws[:0]),
                   dict(dtype=torch.int8), dict(dtype=None)):
        with pytest.raises(RuntimeError):
            gemm.forward(**{**good, **change})
    out = torch.empty(4, 6, dtype=torch.float16, device="cuda")
    for bad in (None, out[:3], out.cpu(), out.int(), out.t(), x.view(torch.float16)[:, :6],
                torch.empty(4, 12, device="cuda").half()[:, ::2]):
        with pytest.raises(RuntimeError):
            gemm.forward_into(**good, out=bad)
    for bad in (None, x, torch.zeros(3, device="cuda"), torch.zeros(3, 4), torch.zeros(
            3, 0, device="cuda"), torch.zeros(3, 4, device="cuda").t()):
        with pytest.raises(RuntimeError):
            gemm.quantize_tokens(bad)
