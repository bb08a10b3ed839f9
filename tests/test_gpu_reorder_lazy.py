"""States that torch keeps as another tensor's memory with a note (conjugate, negative), on an MI355X: their values are gathered."""

from __future__ import annotations

import pytest
import torch

from fie_amd.beam import reorder_states

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_conjugates_and_negatives():
    z = torch.randn(5, 7, dtype=torch.complex64, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    parents = torch.tensor([4, 0, 0, 2, 1], dtype=torch.int32, device=DEV)
    states = [z, z.conj(), z.conj().imag, z.real]
    assert states[1].is_conj() and states[2].is_neg()
    for out in (None, [torch.empty_like(s.resolve_conj().resolve_neg()) for s in states]):
        for s, g in zip(states, reorder_states(states, parents, out=out)):
            assert torch.equal(g, s[parents.long()])
    for lazy, state in ((torch.zeros_like(z).conj(), z), (torch.zeros_like(z).conj().imag, z.real)):
        with pytest.raises(ValueError):
            reorder_states([state], parents, out=[lazy])
