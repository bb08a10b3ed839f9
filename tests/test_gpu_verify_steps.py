"""Verification with token 0 in the contexts: what sample() gives step by step.

The reference's padded scatter undoes token 0's penalty in every row of a step but its widest
(engine/batching/sampler.py:148,156-157,174-175).  A verification's rows are several steps' rows:
those after as many drafts make one step, and a request's later rows, wider by its drafts, are
other steps'."""

from __future__ import annotations

import dataclasses

import numpy as np
import pytest
import torch

import oracle as O
from fie_amd import BatchedSampler, SamplingParams
from fie_amd.verify import DraftVerifier
from test_gpu_verify import LENS, check, make

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_a_draft_after_token_0():
    """Presence 2 takes token 0 from 3.0 to 1.0, below token 8's 2.5, in the draft's row; the row
    after it has 8 in its context as well."""
    x = torch.zeros(2, 16, device=DEV)
    x[:, 0], x[:, 8], x[:, 9] = 3.0, 2.5, 1.5
    s, p = BatchedSampler(DEV), [SamplingParams(presence_penalty=2.0)]
    assert s.sample(x[:1], p, [[0, 5]]).token_ids == [8]
    assert s.sample(x[1:], p, [[0, 5, 8]]).token_ids == [9]
    got = s.verify(x, [[8]], p, context_tokens=[[0, 5]])
    assert got.accepted == [1] and got.token_ids == [[8, 9]]


def test_a_drafted_token_0():
    """Token 0 is drafted, so it is penalised in the rows after it, the last of them the widest."""
    x = torch.zeros(4, 16, device=DEV)
    x[:, 0], x[:, 8], x[:, 9], x[:, 10] = 3.0, 2.5, 2.2, 2.0
    got = BatchedSampler(DEV).verify(x, [[0, 8, 9]], [SamplingParams(presence_penalty=2.0)], context_tokens=[[5]])
    assert got.token_ids == [[0, 8, 9, 10]]


PENALTIES = [dict(presence_penalty=1.5), dict(repetition_penalty=2.0), dict(frequency_penalty=0.7, presence_penalty=0.5)]


@pytest.mark.parametrize("V", [40, 5000])
@pytest.mark.parametrize("requests", [1, 2, 7, 20])
def test_answers_are_those_of_sample_step_by_step(V, requests):
    """Requests that leave nothing to chance (greedy, or one token kept), each of as many drafts:
    the steps of sample() on all of them, the drafts' tokens appended, give every answer."""
    n, rng = 4, np.random.default_rng(V + requests)
    gen = torch.Generator().manual_seed(V + requests)
    x = torch.randn(requests, n + 1, V, generator=gen)
    x[:, :, 0] = 4.0 + 0.2 * torch.randn(requests, n + 1, generator=gen)       # token 0's penalty decides
    x[:, :, 7] = 3.7
    x = x.to(DEV)
    params = [SamplingParams(temperature=(0.0, 0.8)[r % 2], top_k=(0, 1)[r % 2], **PENALTIES[r % 3]) for r in range(requests)]
    contexts = [rng.integers(0, V, 1 + 3 * int(rng.integers(0, 9))).tolist() + [0] * int(r % 4 != 3) for r in range(requests)]
    s = BatchedSampler(DEV, generator_seed=1)
    drafts, steps = [[] for _ in range(requests)], []
    wrong = rng.integers(0, 2 * n, requests)                # a draft that is not the answer, or none
    for j in range(n + 1):
        steps.append(s.sample(x[:, j].contiguous(), params, [c + d for c, d in zip(contexts, drafts)]).token_ids)
        for r in range(requests):
            drafts[r].append((steps[j][r] + int(wrong[r] == j)) % V)
    drafts = [d[:n] for d in drafts]
    want = []
    for r in range(requests):
        k = min(int(wrong[r]), n)
        want.append(drafts[r][:k] + [steps[k][r]])
    got = s.verify(x.view(requests * (n + 1), V), drafts, params, context_tokens=contexts)
    assert got.token_ids == want


def by_place(lens):
    """O.canonical_step on a verification's rows, a step for each number of drafts before them."""
    first = np.cumsum([0] + [n + 1 for n in lens])[:-1]
    places = [np.array([first[r] + j for r in range(len(lens)) if j <= lens[r]]) for j in range(max(lens) + 1)]
    step = O.canonical_step

    def canonical_step(x, res, u, contexts=None, want_kept=False):
        out = step(x, res, u, contexts, want_kept)
        for g in places:
            part = dataclasses.replace(res, **{f.name: getattr(res, f.name)[g] for f in dataclasses.fields(res)
                                               if isinstance(getattr(res, f.name), np.ndarray)})
            one = step(np.asarray(x)[g], part, u[g], None if contexts is None else [contexts[i] for i in g], want_kept)
            for f in dataclasses.fields(out):
                if getattr(out, f.name) is not None:
                    getattr(out, f.name)[g] = getattr(one, f.name)
        return out

    return canonical_step


@pytest.mark.parametrize("V", [300, 9001, 70001])
@pytest.mark.parametrize("requests", [1, 12])
@pytest.mark.parametrize("draft", [None, torch.float32])
def test_ragged_drafts_against_64_bits(monkeypatch, V, requests, draft):
    lens = LENS[:requests] if requests > 1 else [5]
    x, ids, q = make(V + requests, requests, lens, V, torch.float32, draft is not None)
    top = x.amax(1)
    x[:, 0] = top + 0.5                                     # token 0 has a good part of every row
    if q is not None:
        q = 0.7 * q
        q[:, 0] += 0.3
    gen = torch.Generator().manual_seed(V)
    ids = torch.where(torch.rand(len(ids), generator=gen) < 0.4, torch.zeros_like(ids), ids)
    rng = np.random.default_rng(V)
    contexts = [rng.integers(0, V, int(rng.integers(0, 40))).tolist() + [0] * int(r % 3 != 2) for r in range(requests)]
    params = [SamplingParams(temperature=(1.0, 0.7, 0.0, 1.2)[r % 4], top_p=(1.0, 0.9)[r % 2], **PENALTIES[r % 3])
              for r in range(requests)]
    monkeypatch.setattr(O, "canonical_step", by_place(lens))
    check(DraftVerifier(DEV), x, params, lens, ids, q, V + 1, contexts)


def test_ids_outside_the_vocabulary_and_requests_without_penalties():
    """Ids past the vocabulary count in a row's width, rows without penalties do not."""
    V = 32
    x = torch.zeros(3, 3, V, device=DEV)
    x[..., 0], x[..., 8], x[..., 9], x[..., 10] = 3.0, 2.5, 2.2, 2.0
    pen = SamplingParams(presence_penalty=2.0)
    params = [pen, SamplingParams(), pen]
    contexts = [[0, 5], list(range(1, 20)), [V + 3, 0]]
    s = BatchedSampler(DEV)
    drafts = [[8, 9], [0, 0], [8, 9]]
    steps = [s.sample(x[:, j].contiguous(), params, [c + d[:j] for c, d in zip(contexts, drafts)]).token_ids for j in range(3)]
    assert steps[0] == [8, 0, 8] and steps[1][1] == 0
    got = s.verify(x.view(9, V), drafts, params, context_tokens=contexts)
    for r in range(3):
        k = next((j for j in range(2) if steps[j][r] != drafts[r][j]), 2)
        assert got.token_ids[r] == drafts[r][:k] + [steps[k][r]]


def test_more_requests_than_a_workgroup_has_threads():
    """2500 requests of one step after another, their widths all over it, against small batches'
    answers: the widest row of each step alone keeps the penalty, unless ties share it."""
    V, n, R = 300, 2, 2500
    rng = np.random.default_rng(12)
    x = torch.zeros(R, n + 1, V, device=DEV)
    x[..., 0], x[..., 8], x[..., 9], x[..., 10] = 3.0, 2.5, 2.2, 2.0
    pen = SamplingParams(presence_penalty=2.0)
    contexts = [[0] + rng.integers(20, 200, int(rng.integers(0, 30))).tolist() for _ in range(R)]
    contexts[1700] = [0] + list(range(20, 90))              # the widest of all, and again
    contexts[3] = list(contexts[1700])
    drafts = [[8, 9] if r in (3, 1700) or r % 2 else [0, 8] for r in range(R)]
    s = BatchedSampler(DEV)
    steps = [s.sample(x[:, j].contiguous(), [pen] * R, [c + d[:j] for c, d in zip(contexts, drafts)]).token_ids for j in range(n + 1)]
    assert steps[0][3] == steps[0][1700] == 8 and steps[0].count(0) == R - 2
    got = s.verify(x.view(R * (n + 1), V), drafts, [pen] * R, context_tokens=contexts)
    for r in range(R):
        k = next((j for j in range(n) if steps[j][r] != drafts[r][j]), n)
        assert got.token_ids[r] == drafts[r][:k] + [steps[k][r]]
