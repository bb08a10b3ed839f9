"""Totals of beam search are in 64 bits on an MI355X: logits far below their row's largest.

A row's largest logit is `gap` above all others, by 100 and more, so the sum of exp(x - top) is
1 + V * exp(-100) at most, which is 1 in 64 bits, and its logarithm 0: a total is score + (x - top),
both operations exact for the values below (multiples of 2^-20 under 2^12).  In fp32 x - top would have
a unit of 2^-17 and more, and other beams' continuations would tie with it.  Scores come out rounded once.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from fie_amd.beam import beam_step, first_beams

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def best(x, scores, eos, K):
    """(total, beam, token) of the best K that are not in eos: by total, lower beam, larger logit, lower token."""
    total = scores[:, None] + (x - x.max(1, keepdims=True))
    every = [(-total[b, v], b, -x[b, v], v) for b in range(len(x)) for v in range(x.shape[1]) if v not in eos]
    return [(-t, b, v) for t, b, _, v in sorted(every)[:K]]


# the second: more candidates than are ranked at once (64 rows of 80)
@pytest.mark.parametrize("K, V, E", [(4, 60, 1), (64, 200, 16), (9, 20001, 3)])
@pytest.mark.parametrize("gap", [100, 1000, 3000])
def test_far_below_the_largest(K, V, E, gap):
    print(f"  case: {K} x {V}, {E} eos, {gap} below", flush=True)
    gen = torch.Generator().manual_seed(K + gap)
    R, eos = 3, list(range(5, 5 + E))
    # other tokens at multiples of 2^-20 in [0, 2^-14), each row's top an eos that does not exist yet
    x = torch.randint(0, 64, (R * K, V), generator=gen).float() * 2.0 ** -20
    x[:, eos[0]] = gap
    b = first_beams(R, K, DEV)
    b.scores.copy_(-1.0 - torch.randint(0, 8, (R, K), generator=gen) * 2.0 ** -20)
    got = beam_step(x.to(DEV), b, eos=eos, min_tokens=9)
    scores = b.scores.double().cpu().numpy()
    for r in range(R):
        want = best(x[r * K:(r + 1) * K].double().numpy(), scores[r], eos, K)
        assert (got.parents.view(R, K)[r] - r * K).tolist() == [w[1] for w in want]
        assert got.tokens.view(R, K)[r].tolist() == [w[2] for w in want]
        assert got.beams.scores[r].tolist() == [float(np.float32(w[0])) for w in want]
