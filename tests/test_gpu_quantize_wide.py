"""Float tokens and weights as wide as the product takes them (k up to MAX_K)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from fie_amd.linear import MAX_K, int8_linear, quantize_rows

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def plain(x):
    v = x.float().numpy()
    s = np.abs(v).max(1) / np.float32(127)
    with np.errstate(invalid="ignore", divide="ignore"):
        q = np.where(s[:, None] > 0, np.rint(v / s[:, None]), 0)
    return np.nan_to_num(q).astype(np.int8), s


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("width", [65536, 65537, 65543, 100000, 131070, MAX_K])
def test_quantize_rows(dtype, width):
    gen = torch.Generator().manual_seed(width)
    x = torch.randn(7, width, generator=gen).to(dtype)
    x[1] = 0.0
    x[2, width - 1] = 40.0                   # the largest at the row's very end
    x[3, 0] = -40.0
    x[4, 65540 % width] = float("nan")
    x[5] *= 2.0 ** -14
    q, s = quantize_rows(x.to(DEV))
    want_q, want_s = plain(x)
    np.testing.assert_array_equal(s.cpu().numpy(), want_s)
    np.testing.assert_array_equal(q.cpu().numpy()[[0, 1, 2, 3, 5, 6]], want_q[[0, 1, 2, 3, 5, 6]])
    assert np.isnan(want_s[4]) and not q[4].any()
    # a view of a wider storage, at odd addresses
    big = torch.full((7, width + 5), float("nan"), dtype=dtype, device=DEV)
    big[:, 3:3 + width] = x.to(DEV)
    q2, s2 = quantize_rows(big[:, 3:3 + width])
    assert torch.equal(q, q2) and torch.equal(s[[0, 1, 2, 3, 5, 6]], s2[[0, 1, 2, 3, 5, 6]])


@pytest.mark.parametrize("m", [1, 33, 150])
@pytest.mark.parametrize("k", [65537, MAX_K])
def test_products_of_float_tokens(m, k):
    gen = torch.Generator().manual_seed(m + k)
    x, w = torch.randn(m, k, generator=gen), torch.randn(40, k, generator=gen)
    wq, ws = quantize_rows(w.to(DEV))
    got = int8_linear(x.to(DEV), wq, ws).cpu().double()
    (a, sa), (b, sb) = plain(x), plain(w)
    # sums are exact; three fp32 roundings follow them
    want = (torch.from_numpy(a).double() @ torch.from_numpy(b).double().T) * torch.from_numpy(sa).double()[:, None] \
        * torch.from_numpy(sb).double()
    assert ((got - want).abs() <= 4 * 2.0 ** -24 * want.abs()).all()


def test_refusals_name_k():
    w = torch.zeros(2, 8, dtype=torch.int8, device=DEV)
    with pytest.raises(ValueError, match=str(MAX_K)):
        quantize_rows(torch.zeros(1, MAX_K + 1, device=DEV))
    with pytest.raises(ValueError, match=str(MAX_K)):
        int8_linear(torch.zeros(1, MAX_K + 1, device=DEV), w, torch.ones(2, device=DEV))
