"""Products in 8-bit integers on an MI355X against 64 bits.

The sums are exact; (float) of a sum is off by 2^-24 of it, and the two scales and the bias by
as much each: 4 * 2^-24 of |product| + |bias|, then half a unit of the output's type.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from fie_amd.linear import MAX_K, int8_linear, quantize_rows

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def make(seed, m, n, k, full=True):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    lo = -128 if full else -127
    x = torch.randint(lo, 128, (m, k), generator=gen, device=DEV, dtype=torch.int8)
    w = torch.randint(lo, 128, (n, k), generator=gen, device=DEV, dtype=torch.int8)
    xs = torch.rand(m, generator=gen, device=DEV) * 1e-3 + 1e-4
    ws = torch.rand(n, generator=gen, device=DEV) * 1e-3 + 1e-4
    return x, w, xs, ws, torch.randn(n, generator=gen, device=DEV)


def check(got, x, w, xs, ws, bias=None):
    p = (x.double() @ w.double().T) * xs.double()[:, None] * ws.double()
    b = torch.zeros_like(p) if bias is None else bias.double().expand_as(p)
    want = p + b
    bound = HALF[got.dtype] * want.abs() * 1.01 + 4 * 2.0 ** -24 * (p.abs() + b.abs())
    if got.dtype == torch.float16:
        bound = bound + 2.0 ** -25
    off = (got.double() - want).abs()
    bad = off > bound
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float((off / bound).max()))


SIZES = [(1, 1, 1), (1, 16, 64), (1, 4096, 4096), (2, 33, 15), (3, 1000, 17), (5, 64, 128), (7, 65, 129), (16, 4097, 1024),
         (17, 256, 4096), (31, 500, 1003), (33, 2048, 127), (64, 777, 640), (65, 4096, 256), (77, 5001, 1003),
         (100, 130, 2048), (128, 128, 128), (129, 257, 384), (200, 8192, 512), (250, 1024, 4096), (256, 256, 1000),
         (257, 1025, 513), (300, 300, 300), (511, 2000, 1024), (1024, 1024, 1024), (1025, 520, 4096), (2048, 2304, 256),
         (4096, 320, 640)]


@pytest.mark.parametrize("m, n, k", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_sizes(m, n, k, dtype):
    print(f"  case: {m} x {n} x {k} {dtype}", flush=True)
    x, w, xs, ws, bias = make(m * 7 + n + k, m, n, k)
    check(int8_linear(x, w, ws, x_scale=xs, out_dtype=dtype), x, w, xs, ws)
    check(int8_linear(x, w, ws, x_scale=xs, bias=bias, out_dtype=dtype), x, w, xs, ws, bias)


@pytest.mark.parametrize("m", [1, 2, 8, 15, 16, 17, 24, 32, 33, 48, 64, 65, 96, 128, 160, 192, 256, 384, 512, 640])
def test_every_batch_of_a_decode_step(m):
    for n, k in ((4096, 4096), (1536, 8192), (50001, 1024)):
        x, w, xs, ws, _ = make(m, m, n, k)
        check(int8_linear(x, w, ws, x_scale=xs, out_dtype=torch.bfloat16), x, w, xs, ws)


@pytest.mark.parametrize("m", [1, 16, 17, 32, 33, 64, 65, 77, 96, 97, 128, 129])
@pytest.mark.parametrize("n", [4096, 4097, 8193, 9001])
def test_unaligned_rows_of_few_tokens(m, n):
    for k in (1003, 13, 2177):
        x, w, xs, ws, bias = make(m + n + k, m, n, k)
        check(int8_linear(x, w, ws, x_scale=xs, bias=bias, out_dtype=torch.float32), x, w, xs, ws, bias)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_longest_sums_stay_exact(m):
    """The most negative products at the largest k: 2^14 each, just inside 32 bits."""
    x = torch.full((m, MAX_K), -128, dtype=torch.int8, device=DEV)
    w = torch.full((17, MAX_K), -128, dtype=torch.int8, device=DEV)
    w[1] = 127
    w[2, 5] = 0
    one = torch.ones(max(m, 17), device=DEV)
    got = int8_linear(x, w, one[:17], x_scale=one[:m], out_dtype=torch.float32).double()
    want = (x.double() @ w.double().T).float().double()
    assert torch.equal(got, want)


@pytest.mark.parametrize("m, n, k", [(3, 70, 200), (70, 300, 1024), (300, 520, 256), (512, 512, 512)])
def test_strides_and_alignment(m, n, k):
    x, w, xs, ws, _ = make(5, m, n, k)

    def wide(t, pad, at):
        big = torch.full((t.shape[0], t.shape[1] + pad), 77, dtype=t.dtype, device=DEV)
        big[:, at:at + t.shape[1]] = t
        return big, big[:, at:at + t.shape[1]]

    for pad, at in ((3, 1), (16, 0), (32, 16), (128, 64)):
        out, y = wide(torch.zeros(m, n, dtype=torch.float16, device=DEV), pad, at)
        got = int8_linear(wide(x, pad, at)[1], wide(w, pad, at)[1], ws, x_scale=xs, out_dtype=torch.float16, out=y)
        assert got is y
        check(y, x, w, xs, ws)
        assert (out[:, :at] == 77).all() and (out[:, at + n:] == 77).all()
    got = int8_linear(x.t().contiguous().t(), w.t().contiguous().t(), ws, x_scale=xs)
    check(got, x, w, xs, ws)
    check(int8_linear(x[:1].expand(m, k), w, ws, x_scale=xs), x[:1].expand(m, k), w, xs, ws)


def test_float_tokens_are_quantised_first():
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        gen = torch.Generator(device=DEV).manual_seed(1)
        x = torch.randn(3, 11, 500, generator=gen, device=DEV).to(dtype)
        _, w, _, ws, bias = make(2, 1, 90, 500)
        got = int8_linear(x, w, ws, bias=bias)
        assert got.shape == (3, 11, 90) and got.dtype == dtype
        q, s = quantize_rows(x)
        check(got.view(33, 90), q.view(33, 500), w, s, ws, bias)


def test_extreme_scales_and_zero_rows():
    x, w, xs, ws, _ = make(3, 20, 100, 256)
    x[3] = 0
    xs[3] = 0.0
    ws[5] = 0.0
    xs[7] = 1e30
    got = int8_linear(x, w, ws, x_scale=xs, out_dtype=torch.float32)
    assert not got[3].any() and not got[:, 5].any()
    check(got, x, w, xs, ws)


def test_no_tokens_other_streams_and_graphs():
    x, w, xs, ws, _ = make(4, 40, 3000, 2048)
    assert int8_linear(x[:0], w, ws, x_scale=xs[:0]).shape == (0, 3000)
    want = int8_linear(x, w, ws, x_scale=xs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            assert torch.equal(int8_linear(x, w, ws, x_scale=xs), want)
    torch.cuda.current_stream().wait_stream(side)
    for m in (1, 16, 40):
        int8_linear(x[:m], w, ws, x_scale=xs[:m])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        y = torch.empty(m, 3000, dtype=torch.bfloat16, device=DEV)
        xin = x[:m].clone()
        with torch.cuda.graph(graph):
            int8_linear(xin, w, ws, x_scale=xs[:m], out=y)
        for i in range(4):
            xin.copy_(torch.roll(x[:m], i + 1, 1))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, int8_linear(xin, w, ws, x_scale=xs[:m]))


def test_large_offsets():
    """Weights past 2^31 bytes: 140000 channels of 16384, the last ones checked."""
    n, k = 140000, 16384
    w = torch.zeros((n, k), dtype=torch.int8, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(6)
    w[-300:] = torch.randint(-127, 128, (300, k), generator=gen, device=DEV, dtype=torch.int8)
    x = torch.randint(-127, 128, (130, k), generator=gen, device=DEV, dtype=torch.int8)
    one = torch.full((n,), 1e-3, device=DEV)
    for m in (1, 20, 130):
        got = int8_linear(x[:m], w, one, x_scale=one[:m], out_dtype=torch.float32)
        check(got[:, -300:], x[:m], w[-300:], one[:m], one[:300])
        assert not got[:, :1000].any()


def test_refusals():
    x, w, xs, ws, bias = make(9, 4, 32, 64)
    good = dict(x=x, weight=w, weight_scale=ws, x_scale=xs)
    for bad in (dict(x=x[:, :63]), dict(x_scale=None), dict(x_scale=xs[:3]), dict(x_scale=xs.half()), dict(weight_scale=ws[:31]),
                dict(weight=w.float()), dict(weight=w[0]), dict(bias=bias[:5]), dict(bias=bias.half()), dict(x=x.double()),
                dict(x=x.float()), dict(out_dtype=torch.int8), dict(out=torch.empty(4, 32, device=DEV)), dict(x=x.cpu()),
                dict(weight=w.cpu()), dict(out=torch.empty(3, 32, dtype=torch.bfloat16, device=DEV)),
                dict(out=torch.empty(32, 4, dtype=torch.bfloat16, device=DEV).t()), dict(weight_scale=torch.cat([ws, ws])[::2]),
                dict(x=x[:, :0], weight=w[:, :0])):
        kw = {**good, **bad}
        with pytest.raises(ValueError):
            int8_linear(kw.pop("x"), kw.pop("weight"), kw.pop("weight_scale"), **kw)
    big = torch.empty(1, MAX_K + 1, dtype=torch.int8, device=DEV)
    with pytest.raises(ValueError):
        int8_linear(big, big, xs[:1], x_scale=xs[:1])
    np.testing.assert_equal(MAX_K * 128 * 128 < 2 ** 31, True)
