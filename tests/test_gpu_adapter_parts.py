"""Adapters in fp16 on an MI355X whose ranks are of very different size: h = A x enters the second product
as two fp16 numbers, brought by a power of two to a largest |h| of m in [2^14, 2^15).

The leading part is off by 2^-11 |h|, the rest is exact in fp32, and the trailing part rounds the rest by
2^-11 of it, 2^-22 |h|, or, where that is below fp16's normal numbers, by half of 2^-24, which is at
most 2^-39 m.  (A leading part below them leaves a rest of 2^-25 or less, rounded by no more than itself.)

Tokens have one element that is not 0 and channels one rank, so h is one exact product of two fp16 numbers
and y the sum of two more, rounded by 2^-24 at each of: either product, their sum, a token's scale in
the factor, the factor's product.
"""

from __future__ import annotations

import pytest
import torch

from fie_amd.adapters import AdapterBank, adapter_linear
from fie_amd.linear import quantize_rows

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
UNIT = 2.0 ** -24


@pytest.mark.parametrize("rank", [16, 13, 48, 64, 80])
@pytest.mark.parametrize("size", [1.0, 2.0 ** -9, 2.0 ** 9])
def test_ranks_of_very_different_size(rank, size):
    """A's row j times 2^-j (of 16), B's column j times 2^j."""
    tokens, k, n = 40, 64, 200
    gen = torch.Generator(device=DEV).manual_seed(rank)

    def rnd(*s):                                        # in (-1, -1/2] and [1/2, 1)
        v = torch.rand(*s, generator=gen, device=DEV) - 0.5
        return v + torch.where(v < 0, -0.5, 0.5)

    step = 2.0 ** -(torch.arange(rank, device=DEV) % 16).float()
    a = (rnd(rank, k) * step[:, None]).half()
    b = (rnd(n, rank) / step).half() * (torch.arange(n, device=DEV)[:, None] % rank == torch.arange(rank, device=DEV))
    bank = AdapterBank(1, k, n, rank, torch.float16, DEV)
    bank.load(0, a, b, 1.0)
    plan = bank.plan(torch.zeros(tokens, dtype=torch.int32, device=DEV))
    x = (size * rnd(tokens, k) * (torch.arange(tokens, device=DEV)[:, None] == torch.arange(k, device=DEV))).half()
    q, s = quantize_rows(x)
    for got, x in ((adapter_linear(x, bank, plan, out_dtype=torch.float32), x.double()),
                   (adapter_linear(q, bank, plan, x_scale=s, out_dtype=torch.float32), q.double() * s.double()[:, None])):
        h = x @ a.double().T
        off = torch.maximum(2.0 ** -22 * h.abs(), 2.0 ** -39 * h.abs().amax(1, keepdim=True)) @ b.double().abs().T
        want = h @ b.double().T
        bad = (got.double() - want).abs() > off + 5 * UNIT * (want.abs() + off)
        assert want.abs().min() > 0 and not bad.any(), (int(bad.sum()), float(((got.double() - want) / want).abs().max()))
