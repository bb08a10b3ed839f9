"""NaN and infinities through the quantisation and the product behind it: a broken activation
stays visible in the logits of its own token, and of no other."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from fie_amd.linear import int8_linear, quantize_rows
from fie_amd.norm import block_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NAN, INF = float("nan"), float("inf")


def tokens(width, dtype, rows=6, seed=1):
    gen = torch.Generator().manual_seed(seed + width)
    return torch.randn(rows, width, generator=gen).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("width", [1, 2, 9, 17, 64, 1000, 4096, 16385, 65536])
def test_a_row_with_nan_has_a_nan_scale(dtype, width):
    x = tokens(width, dtype)
    want_q, want_s = quantize_rows(x.to(DEV))
    scale = np.abs(x.float().numpy()).max(1) / np.float32(127)
    np.testing.assert_array_equal(want_s.cpu().numpy(), scale)
    np.testing.assert_array_equal(want_q.cpu().numpy(), np.rint(x.float().numpy() / scale[:, None]).astype(np.int8))
    sign = torch.tensor([1.0, -1.0])[:, None] * torch.tensor(NAN)
    for at in sorted({0, width // 2, width - 1}):
        y = x.clone()
        y[1, at], y[4, at] = sign[0, 0], sign[1, 0]
        y[4, 0] = NAN
        q, s = quantize_rows(y.to(DEV))
        assert torch.isnan(s[[1, 4]]).all()
        assert not q[[1, 4]].any()
        rest = [0, 2, 3, 5]
        assert torch.equal(q[rest], want_q[rest]) and torch.equal(s[rest], want_s[rest])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("width", [1, 17, 64, 1000, 4096, 16385])
def test_quantize_rows_is_the_ieee_quotient(dtype, width):
    gen = torch.Generator().manual_seed(width)
    x = (torch.randn(6, width, generator=gen) * torch.tensor([1.0, 1e-3, 300.0, 1e-7, 0.0, 50.0])[:, None]).to(dtype)
    x[5, 0] = NAN
    q, s = quantize_rows(x.to(DEV))
    v = x.float().numpy()
    want = np.abs(v).max(1) / np.float32(127)               # NaN where the row has one
    assert np.isnan(want[5]) and want[4] == 0
    np.testing.assert_array_equal(s.cpu().numpy(), want)
    with np.errstate(invalid="ignore", divide="ignore"):
        t = np.rint(v / want[:, None])
    np.testing.assert_array_equal(q.cpu().numpy(), np.where(np.isnan(t), 0, t).astype(np.int8))


@pytest.mark.parametrize("kind", ["rms", "layer", "none"])
@pytest.mark.parametrize("width", [5, 512, 1003, 4096, 20000])
@pytest.mark.parametrize("value", [NAN, -NAN, INF, -INF])
def test_block_norm_to_int8_and_its_product(kind, width, value):
    x = tokens(width, torch.bfloat16, rows=5).to(DEV)
    r = tokens(width, torch.bfloat16, rows=5, seed=7).to(DEV)
    wq, ws = quantize_rows(tokens(width, torch.float32, rows=70, seed=9).to(DEV))
    clean = block_norm(r, x, kind=kind, quantize=True)
    x[2, width // 3] = value
    got = block_norm(r, x, kind=kind, quantize=True)
    logits = int8_linear(got.y, wq, ws, x_scale=got.scale, out_dtype=torch.float32)
    plain = int8_linear(clean.y, wq, ws, x_scale=clean.scale, out_dtype=torch.float32)
    if kind != "none" or value != value:
        assert torch.isnan(got.scale[2])
    assert torch.isnan(logits[2]).all()
    rest = [0, 1, 3, 4]
    assert torch.equal(got.y[rest], clean.y[rest]) and torch.equal(got.scale[rest], clean.scale[rest])
    assert torch.equal(logits[rest], plain[rest])


@pytest.mark.parametrize("m, k", [(1, 64), (16, 1003), (70, 256), (200, 1003), (300, 4096)])
@pytest.mark.parametrize("bias", [False, True])
def test_float_tokens_with_nan(m, k, bias):
    x = tokens(k, torch.float16, rows=m).to(DEV)
    wq, ws = quantize_rows(tokens(k, torch.float32, rows=90, seed=9).to(DEV))
    b = torch.ones(90, device=DEV) if bias else None
    plain = int8_linear(x, wq, ws, bias=b)
    x[m // 2, k - 1] = NAN
    got = int8_linear(x, wq, ws, bias=b)
    assert torch.isnan(got[m // 2]).all()
    rest = torch.arange(m, device=DEV) != m // 2
    assert torch.equal(got[rest], plain[rest])


def test_a_channel_with_nan():
    w = tokens(128, torch.float32, rows=40, seed=3).to(DEV)
    w[11, 100] = NAN
    wq, ws = quantize_rows(w)
    y = int8_linear(tokens(128, torch.float32).to(DEV), wq, ws)
    assert torch.isnan(y[:, 11]).all()
    assert torch.isfinite(y[:, [c for c in range(40) if c != 11]]).all()
