"""Totals below the least fp32 number on an MI355X: they are held at it, since -inf says that no beam
is there.  A logit of +inf counts as the largest fp32 number, so a token at the type's lowest value beside it
is twice that below; and an answer's value is its total over a power that may be far below 1."""

from __future__ import annotations

import pytest
import torch

from fie_amd.beam import beam_step, first_beams

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
LOWEST = torch.finfo(torch.float32).min


def only(R, K, V, dtype):
    """One request a row of logits, at its first step."""
    return torch.full((R * K, V), float("-inf"), device=DEV).to(dtype), first_beams(R, K, DEV)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [5, 9000])
def test_the_lowest_value_exists_beside_an_infinity(V, dtype):
    K, low = 4, torch.finfo(dtype).min
    x, b = only(2, K, V, dtype)
    x[0, [1, 2, V - 1]] = low
    x[0, 0] = float("inf")
    x[K, 0] = float("inf")                              # and nothing else: one beam
    got = beam_step(x, b)
    assert got.tokens[:K].tolist() == [0, 1, 2, V - 1] and got.parents[:K].tolist() == [0] * K
    assert got.beams.scores[0].tolist() == [0.0, LOWEST, LOWEST, LOWEST]
    assert got.beams.scores[1].tolist() == [0.0] + [float("-inf")] * 3 and got.tokens[K + 1:].tolist() == [0] * 3
    assert not got.beams.done.any()
    # they go on from there: total LOWEST - log 2, of which LOWEST's unit (2^104) leaves LOWEST
    x, _ = only(2, K, V, dtype)
    x[:K, :2] = 1.0
    got = beam_step(x, got.beams)
    assert got.parents[:K].tolist() == [0, 0, 1, 1] and got.tokens[:K].tolist() == [0, 1, 0, 1]
    assert got.beams.scores[0, 2:].tolist() == [LOWEST, LOWEST] and got.beams.lengths.tolist() == [2, 2]
    assert got.beams.done.tolist() == [False, True]     # the other request has no logits left


def test_an_answer_of_such_a_total():
    K, V = 2, 6
    x, b = only(1, K, V, torch.float32)
    x[0, 0], x[0, 3] = float("inf"), LOWEST
    got = beam_step(x, b, eos=[3])
    assert got.tokens.tolist() == [0, 0] and got.beams.pool.tolist() == [[LOWEST, float("-inf")]]
    assert got.beams.ends[0, 0].tolist() == [1, 0, 3]
    # a total of -log 2 over 2 ^ -200 is below LOWEST, too
    x, b = only(1, K, V, torch.float32)
    x[0, :2] = 0.0
    b.lengths.fill_(1)
    got = beam_step(x, b, eos=[1], length_penalty=-200.0)
    assert got.beams.pool.tolist() == [[LOWEST, float("-inf")]] and got.beams.ends[0, 0].tolist() == [2, 0, 1]
