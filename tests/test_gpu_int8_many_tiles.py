"""8-bit products of more tiles than one launch holds (2^32 threads)."""

from __future__ import annotations

import pytest
import torch

from fie_amd.linear import int8_linear

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def operands(rows, k, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randint(-127, 128, (rows, k), dtype=torch.int8, generator=gen, device=DEV),
            0.5 + torch.rand(rows, generator=gen, device=DEV))


@pytest.mark.parametrize("k", [16, 5])
def test_many_tokens(k):
    """2^23 tiles of 32 tokens, 512 threads each, and some; rows at 16 bytes, and laid out first."""
    m, n = 2 ** 28 + 37, 7
    x, xs = operands(m, k, 1)
    w, ws = operands(n, k, 2)
    got = int8_linear(x, w, ws, x_scale=xs)
    step = 2 ** 24
    for at in (0, step - 20, 2 ** 27, m - 90):
        part = slice(at, at + 90)
        assert bool((got[part] == int8_linear(x[part], w, ws, x_scale=xs[part])).all())
    # every row, against the plain product (its sums are whole numbers below 2^24)
    for at in range(0, m, step):
        part = slice(at, min(at + step, m))
        want = (x[part].float() @ w.float().T) * xs[part, None] * ws
        assert bool((got[part] == want.bfloat16()).all())


@pytest.mark.parametrize("m", [3, 40])
def test_many_channels(m):
    """Channels past one launch of either kernel's (rows at 16 bytes and not)."""
    n = 2 ** 28 + 75
    for k in (16, 5):
        x, xs = operands(m, k, 3)
        w, ws = operands(n, k, 4)
        bias = torch.rand(n, device=DEV)
        got = int8_linear(x, w, ws, x_scale=xs, bias=bias)
        for at in list(range(0, n - 100, 2 ** 25 - 31)) + [n - 100]:
            part = slice(at, at + 100)
            want = (x.float() @ w[part].float().T) * xs[:, None] * ws[part] + bias[part]
            assert bool((got[:, part] == want.bfloat16()).all())
        del w, ws, bias, got
