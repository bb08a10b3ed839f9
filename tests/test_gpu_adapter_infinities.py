"""Tokens with infinite activations through adapters on an MI355X: the result is the formula's, an infinity or no number,
whatever the adapter's rank is padded to.  All other tokens keep their bits."""

from __future__ import annotations

import pytest
import torch

from fie_amd.adapters import AdapterBank, adapter_linear

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rank, room", [(1, 1), (1, 16), (3, 20), (16, 16), (16, 40), (17, 17), (33, 33), (50, 64), (1, 100), (70, 100)])
def test_infinite_activations(rank, room, dtype):
    tokens, k, n = 37, 130, 70
    gen = torch.Generator(device=DEV).manual_seed(rank + room)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    a, b, x = rnd(rank, k), rnd(n, rank), rnd(tokens, k).to(dtype)
    # one sign a column of A, one a row of B: infinities of one sign meet
    a[:, 5] = a[:, 5].abs() + 0.1
    a[:, 129] = -a[:, 129].abs() - 0.1
    b = (b.abs() + 0.1) * torch.where(rnd(n, 1) > 0, 1.0, -1.0)
    a, b = a.to(dtype), b.to(dtype)
    bank = AdapterBank(2, k, n, room, dtype, DEV)
    bank.load(1, a, b, 0.5)
    ids = torch.ones(tokens, dtype=torch.int32, device=DEV)
    ids[::5] = -1
    base = rnd(tokens, n).to(dtype)
    plan = bank.plan(ids)
    clean = adapter_linear(x, bank, plan, base=base)
    x[2, 5], x[3, 129], x[4, 5], x[7, 5], x[8, 0] = float("inf"), float("inf"), float("-inf"), float("inf"), float("nan")
    x[7, 129] = float("inf")                            # against the other: no number
    x[5, 5] = float("inf")                              # a token without an adapter
    got = adapter_linear(x, bank, plan, base=base)
    want = base.double() + 0.5 * ((x.double() @ a.double().T) @ b.double().T)
    for t in (2, 3, 4):
        assert torch.isinf(want[t]).all() and torch.equal(got[t].double(), want[t]), t
    for t in (7, 8):
        assert want[t].isnan().all() and got[t].isnan().all(), t
    other = [t for t in range(tokens) if t not in (2, 3, 4, 7, 8)]
    assert torch.equal(got[other], clean[other])
