"""BatchedSampler.verify() and the example that runs the operators together, on an MI355X."""

from __future__ import annotations

import importlib.util
import os

import numpy as np
import pytest
import torch

from fie_amd import BatchedSampler, SamplingParams
from fie_amd.batching.sampler import SEEDED_STREAM
from fie_amd.verify import DraftVerifier

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def batch(seed, lens, V):
    gen = torch.Generator().manual_seed(seed)
    x = 2.0 * torch.randn(sum(lens) + len(lens), V, generator=gen)
    ids = torch.randint(0, V, (sum(lens),), generator=gen)
    q = torch.softmax(torch.randn(sum(lens), V, generator=gen), 1)
    drafts, at = [], 0
    for n in lens:
        drafts.append(ids[at:at + n].tolist())
        at += n
    return x.to(DEV), drafts, q.to(DEV), ids.to(DEV)


def test_greedy_requests_keep_their_argmax():
    V = 500
    x, drafts, _, _ = batch(1, [3, 2, 0, 4], V)
    top = x.argmax(1).tolist()
    drafts = [top[0:3], [top[4], (top[5] + 1) % V], [], top[8:10] + [0, 0]]
    got = BatchedSampler(DEV).verify(x, drafts, [SamplingParams()] * 4)
    assert got.accepted == [3, 1, 0, 2 if top[10] else 3]
    assert got.token_ids[0] == top[0:4]
    assert got.token_ids[1] == [top[4], top[5]]
    assert got.token_ids[2] == [top[7]]
    assert got.token_ids[3][:3] == top[8:11]


def test_seeded_requests_draw_their_own_stream():
    V, lens = 3000, [2, 3, 1]
    x, drafts, q, ids = batch(2, lens, V)
    params = [SamplingParams(temperature=1.0, seed=5), SamplingParams(temperature=0.8, top_p=0.9, seed=9), SamplingParams()]
    s = BatchedSampler(DEV, generator_seed=1)
    first = s.verify(x, drafts, params, q, request_ids=["a", "b", "c"])
    second = s.verify(x, drafts, params, q, request_ids=["a", "b", "c"])
    v = DraftVerifier(DEV)
    for step, got in enumerate((first, second)):
        rng = np.zeros((sum(lens) + 3, 3), np.uint64)
        rng[:3] = [[5, SEEDED_STREAM, 3 * step + 1 + j] for j in range(3)]
        rng[3:7] = [[9, SEEDED_STREAM, 4 * step + 1 + j] for j in range(4)]
        want = v.verify(v.plan(params, lens, V, rng=rng), x, ids, None, q)
        assert got.accepted == want.accepted.tolist()
        assert got.token_ids == [r[:n + 1] for r, n in zip(want.tokens.tolist(), got.accepted)]
    # alone and in another order: the same tokens
    t = BatchedSampler(DEV, generator_seed=77)
    alone = t.verify(x[3:7], [drafts[1]], [params[1]], q[2:5], request_ids=["b"])
    assert alone.token_ids[0] == first.token_ids[1]
    t.forget(["b"])
    again = t.verify(x[3:7], [drafts[1]], [params[1]], q[2:5], request_ids=["b"])
    assert again.token_ids == alone.token_ids


def test_without_drafts_it_samples():
    """No drafts: the tokens of sample() on the same streams."""
    V, R = 5000, 40
    x = 2.0 * torch.randn(R, V, device=DEV, generator=torch.Generator(device=DEV).manual_seed(3))
    params = [SamplingParams(temperature=0.5 + 0.05 * (i % 7), top_k=(0, 20)[i % 2], seed=i) for i in range(R)]
    a, b = BatchedSampler(DEV), BatchedSampler(DEV)
    got = a.verify(x, [[]] * R, params)
    assert [t for row in got.token_ids for t in row] == b.sample(x, params).token_ids
    # and after it, sample() goes on in the stream
    assert a.sample(x, params).token_ids == b.sample(x, params).token_ids


def test_penalties_see_the_drafts():
    """A drafted token counts in the rows after it: greedy with a large presence penalty never
    keeps the same token twice."""
    V = 200
    x = torch.zeros(4, V, device=DEV)
    x[:, 7], x[:, 8], x[:, 9] = 3.0, 2.5, 2.0
    params = [SamplingParams(presence_penalty=2.0)]
    got = BatchedSampler(DEV).verify(x, [[7, 8, 7]], params, context_tokens=[[1, 2]])
    assert got.token_ids == [[7, 8, 9]] and got.accepted == [2]


def test_refusals():
    x, drafts, q, _ = batch(4, [1, 2], 64)
    s, p = BatchedSampler(DEV), [SamplingParams(temperature=1.0)] * 2
    assert s.verify(x[:0], [], []).token_ids == []
    for args in ((x[0], drafts, p), (x[:4], drafts, p), (x, drafts, p[:1]), (x, [[64], [1, 2]], p), (x, [[-1], [1, 2]], p),
                 (x, drafts, p, q[:2]), (x, drafts, p, q, [[1]]), (x, drafts, p, q, None, ["a"]),
                 (x, drafts, [SamplingParams(logprobs=2)] * 2), (x.cpu(), drafts, p)):
        with pytest.raises(ValueError):
            s.verify(*args)


def test_the_example_runs_and_keeps_drafts():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "speculative_step.py")
    spec = importlib.util.spec_from_file_location("speculative_step", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    good = example.run(requests=6, drafts=3, steps=8, vocab=4000, hidden=256, noise=0.05)
    bad = example.run(requests=6, drafts=3, steps=8, vocab=4000, hidden=256, noise=3.0)
    assert good["new_tokens"] == 6 * 8 * good["tokens_per_step"] >= 6 * 8
    assert all(0 <= t < 4000 for o in good["outputs"] for t in o)
    assert good["kept_share"] > 0.8 > bad["kept_share"]
