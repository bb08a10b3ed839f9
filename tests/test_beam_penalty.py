"""Length penalties that are no finite number are refused, and finite ones whose power leaves the doubles
give values all the same: refusals and a search's answers on the CPU, the pool on an MI355X."""

from __future__ import annotations

import struct

import pytest
import torch

from fie_amd import _lib, beam
from fie_amd.beam import BeamSearch, Beams, beam_step, first_beams

INF = float("inf")
LOWEST = torch.finfo(torch.float32).min


class OnDevice(torch.Tensor):
    """A host tensor that says it is on device 0."""

    def get_device(self):
        return 0


@pytest.mark.parametrize("penalty", [INF, -INF, float("nan")])
def test_refused_by_the_library(penalty):
    names = 13 * [256] + [0, 0, 100, 256, 1 << 20, penalty, 2, 4, 100] + 6 * [0] + 16 * [0] + [0]
    lib = _lib.load()
    assert lib.fie_beam_step(struct.pack(_lib.BEAM_ARGS, *names), None) == _lib.FIE_E_ARG
    assert b"length_penalty" in lib.fie_sampler_last_error()


@pytest.mark.parametrize("penalty", [INF, -INF, float("nan")])
def test_refused_by_the_call(monkeypatch, penalty):
    calls = []
    monkeypatch.setattr(beam, "_run", lambda *a: calls.append(a))
    monkeypatch.setattr(beam, "_size", lambda a: 64)
    b = Beams(*(t.as_subclass(OnDevice) for t in first_beams(2, 3, "cpu")))
    x = torch.zeros(6, 10).as_subclass(OnDevice)
    beam_step(x, b, length_penalty=-3.5)
    assert len(calls) == 1
    with pytest.raises(ValueError, match="length_penalty"):
        beam_step(x, b, length_penalty=penalty)
    assert len(calls) == 1


def test_answers_of_extreme_penalties():
    """score / length ** penalty of beams that are still searched, length 2."""
    search = BeamSearch.__new__(BeamSearch)
    search.requests, search.count, search.max_tokens = 1, 2, 4
    search.beams = first_beams(1, 2, "cpu")
    search.beams.scores.copy_(torch.tensor([[0.0, -3.0]]))
    search.beams.lengths.fill_(2)
    search._history = torch.tensor([[5, 6], [7, 8], [0, 0], [0, 0]]).int(), torch.tensor([[0, 0], [0, 1], [0, 0], [0, 0]]).int()
    for penalty, want in ((1.0, [0.0, -1.5]), (1e4, [0.0, 0.0]), (-1e4, [0.0, LOWEST]), (-200.0, [0.0, LOWEST])):
        search._settings = dict(length_penalty=penalty)
        got = search.answers(0)
        assert [a.value for a in got] == want and [a.tokens for a in got] == [[5, 7], [6, 8]]


DEV = "cuda:0"


@pytest.mark.gpu
@pytest.mark.parametrize("penalty, value", [(1e4, 0.0), (800.0, 0.0), (-800.0, LOWEST), (-1e4, LOWEST), (-1e300, LOWEST), (1e300, 0.0)])
def test_pool_of_extreme_penalties(penalty, value):
    """Two endings of total -log 2 and, of another request, one of total 0, at length 2."""
    K, V = 3, 9
    x = torch.full((2 * K, V), -INF, device=DEV)
    x[0, [1, 2]] = 0.0
    x[K, 2] = 4.0
    b = first_beams(2, K, DEV)
    b.lengths.fill_(1)
    got = beam_step(x, b, eos=[1, 2], length_penalty=penalty).beams
    assert got.done.all() and got.lengths.tolist() == [2, 2]
    assert got.ends.tolist() == [[[2, 0, 1], [2, 0, 2], [-1] * 3], [[2, K, 2], [-1] * 3, [-1] * 3]]
    assert got.pool.tolist() == [[value, value, -INF], [0.0, -INF, -INF]]
    # and an older answer stays where its value puts it
    b.pool[0, 0] = -7.0
    b.ends[0, 0] = 5
    got = beam_step(x, b, eos=[1, 2], length_penalty=penalty).beams
    assert sorted(got.pool[0].tolist(), reverse=True) == got.pool[0].tolist() and -7.0 in got.pool[0].tolist()


@pytest.mark.gpu
def test_penalties_of_the_first_token():
    """1 to any power: the total itself."""
    K, V = 2, 5
    x = torch.full((K, V), -INF, device=DEV)
    x[0, [1, 2]] = 0.0
    for penalty in (-1e300, -2.5, 0.0, 1.0, 3.0, 1e300):
        got = beam_step(x, first_beams(1, K, DEV), eos=[1, 2], length_penalty=penalty).beams
        torch.testing.assert_close(got.pool, torch.full((1, K), -0.6931472, device=DEV), rtol=0, atol=2e-6)
