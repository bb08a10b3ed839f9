"""Block norms of more rows than one launch holds (2^32 threads): narrow heads of a long batch."""

from __future__ import annotations

import pytest
import torch

from fie_amd.linear import quantize_rows
from fie_amd.norm import block_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROWS = 2 ** 26 + 9                           # a wave a row: 2^32 threads and some


@pytest.mark.parametrize("gate", [None, "row"])
def test_more_rows_than_a_launch_holds(gate):
    gen = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn(ROWS, 8, generator=gen, device=DEV).half()
    w = torch.randn(8, generator=gen, device=DEV).half()
    g = torch.rand(ROWS, 1, generator=gen, device=DEV).half() if gate else None
    got = block_norm(x, x, w, gate=g, scale=0.5)
    for at in (0, 2 ** 25, 2 ** 26 - 40, 2 ** 26 - 4):              # each end of the pieces
        part = slice(at, at + 64)
        one = block_norm(x[part], x[part], w, gate=None if g is None else g[part], scale=0.5)
        assert torch.equal(got.y[part], one.y) and torch.equal(got.residual[part], one.residual)


def test_more_rows_quantised_than_a_launch_holds():
    gen = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(ROWS, 5, generator=gen, device=DEV).bfloat16()
    q, s = quantize_rows(x)
    for at in (0, 2 ** 25, 2 ** 26 - 40, 2 ** 26 - 4):
        part = slice(at, at + 64)
        want = quantize_rows(x[part])
        assert torch.equal(q[part], want[0]) and torch.equal(s[part], want[1])
