"""Exactly equal totals on an MI355X: by the lower beam, then the larger logit, then the lower token, and
no continuation twice.

Rows of V logits whose bytes are a multiple of 16 are summed in the same order wherever they are, so
equal rows have bit-equal sums, and equal beams with equal rows exactly equal totals.
"""

from __future__ import annotations

import pytest
import torch

from fie_amd.beam import beam_step, first_beams

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def alive(R, K, score=-1.0):
    b = first_beams(R, K, DEV)
    b.scores.fill_(score)
    return b


def distinct(got):
    """No continuation of a request twice (rows that go on; others have themselves as parent)."""
    R, K = got.beams.scores.shape
    for r in range(R):
        on = torch.isfinite(got.beams.scores[r]).tolist()
        pairs = [p for p, o in zip(zip(got.parents[r * K:].tolist(), got.tokens[r * K:].tolist()), on) if o]
        assert len(set(pairs)) == len(pairs), r


# the last three: more candidates than one ranking takes, or than its list holds
@pytest.mark.parametrize("R, K, V, eos", [(1, 1, 8, []), (3, 4, 1000, [1]), (2, 16, 60000, [0, 2]), (1, 64, 151936, [0, 1, 3, 151935]),
                                          (2, 40, 100000, [5]), (1, 64, 256, list(range(1, 17)))])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_constant_logits(R, K, V, eos, dtype):
    """Every total alike: the lowest tokens of the lowest beam."""
    print(f"  case: {R} x {K} x {V} {dtype}", flush=True)
    want = [v for v in range(V) if v not in eos][:K]
    for value in (0.0, 1.0, -3.5):
        got = beam_step(torch.full((R * K, V), value, device=DEV).to(dtype), alive(R, K), eos=eos)
        assert got.tokens.view(R, K).tolist() == [want] * R
        assert got.parents.view(R, K).tolist() == [[r * K] * K for r in range(R)]
        # those that end: the eos among the first K of the lowest beam
        ended = [v for v in range(K) if v in eos]
        ends = got.beams.ends[:, :len(ended)].tolist()
        assert ends == [[[1, r * K, v] for v in ended] for r in range(R)]


@pytest.mark.parametrize("R, K, V", [(2, 4, 2000), (3, 16, 60000), (1, 64, 8192), (2, 33, 40000)])
def test_equal_beams(R, K, V):
    """The same row for every beam: each of its values K times over, the beams in order."""
    print(f"  case: {R} x {K} x {V}", flush=True)
    gen = torch.Generator().manual_seed(V)
    for levels in (3, 40, 5000):                                        # of the logits: many ties, some, few
        x = (torch.randint(0, levels, (1, V), generator=gen).half() * (8.0 / levels)).to(DEV)
        eos = [7, V - 1]
        got = beam_step(x.expand(R * K, V), alive(R, K), eos=eos)
        value = x[0].float().cpu()
        value[eos] = float("-inf")
        top = (value == value.max()).nonzero()[:, 0].tolist()
        # beam 0 has all of its best tokens in front of beam 1's, and so on
        want = [(b, v) for b in range(K) for v in top][:K]
        if len(want) == K:
            assert [(p - r * K, t) for r in range(R) for p, t in zip(got.parents.view(R, K)[r].tolist(), got.tokens.view(R, K)[r].tolist())] \
                == want * R
        distinct(got)


@pytest.mark.parametrize("R, K, V, E", [(4, 4, 1000, 1), (1, 64, 50001, 16), (2, 40, 100001, 3), (30, 8, 9001, 2), (3, 5, 12, 4)])
@pytest.mark.parametrize("spread", [0.0, 0.01, 3.0])
def test_no_continuation_twice(R, K, V, E, spread):
    gen = torch.Generator(device=DEV).manual_seed(V + K)
    x = (spread * torch.randn(R * K, V, generator=gen, device=DEV)).bfloat16()
    b = alive(R, K)
    for _ in range(3):
        got = beam_step(x, b, eos=list(range(E)))
        distinct(got)
        b = got.beams
