"""A refused verification takes no draws: called again correctly, it answers as if the refused
call had not been made."""

from __future__ import annotations

import pytest
import torch

from fie_amd import BatchedSampler, SamplingParams
from fie_amd.batching import sampler
from fie_amd.verify import MAX_DRAFTS

DEV = "cuda:0"


def test_refusals_before_anything_is_uploaded_take_no_draws(monkeypatch):
    V = 50
    x = torch.zeros(2, V)
    one = [SamplingParams(temperature=1.0, seed=3)]
    monkeypatch.setattr(sampler, "DeviceHistory", lambda device: None)      # its store is on the device
    s = BatchedSampler(DEV, generator_seed=3)
    for args in ((x, [[3]], [SamplingParams(temperature=1.0, logprobs=0)]),
                 (torch.zeros(MAX_DRAFTS + 2, V), [[1] * (MAX_DRAFTS + 1)], one),
                 (x, [[3]], [SamplingParams(temperature=1.0, presence_penalty=1.0)], None, [[4, -1]]),
                 (x, [[3]], [SamplingParams(temperature=1.0, presence_penalty=1.0, seed=2)], None, [[2 ** 31]])):
        with pytest.raises(ValueError):
            s.verify(*args)
        assert s._shared_draws == 0 and not s._seeded


@pytest.mark.gpu
def test_refused_calls_take_no_draws():
    V = 500
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(5, V, generator=gen).to(DEV)
    q = torch.softmax(torch.randn(3, V, generator=gen), 1).to(DEV)
    drafts, ids = [[3], [4, 5]], ["a", "b"]
    params = [SamplingParams(temperature=1.0, seed=7), SamplingParams(temperature=1.0)]
    pen = [SamplingParams(temperature=1.0, seed=7, presence_penalty=1.0), params[1]]
    long = torch.zeros(MAX_DRAFTS + 2, V, device=DEV)
    s, fresh = BatchedSampler(DEV, generator_seed=3), BatchedSampler(DEV, generator_seed=3)
    assert s.verify(x, drafts, params, q, request_ids=ids) == fresh.verify(x, drafts, params, q, request_ids=ids)
    counters = (s._shared_draws, dict(s._seeded))
    for args in ((x, drafts, params, q[:2]), (x, drafts, params, q[:, :99]), (x, drafts, params, q.double()),
                 (x, drafts, params, q.cpu()), (x.cpu(), drafts, params, q), (x[0], drafts, params),
                 (x, drafts, [SamplingParams(temperature=1.0, logprobs=2)] * 2), (x, drafts, params[:1]),
                 (long, [[1] * (MAX_DRAFTS + 1)], params[:1]), (x, [[V], [4, 5]], params),
                 (x, drafts, pen, q, [[1, -5], [2]]), (x, drafts, params, q, [[1]]), (x, drafts, params, q, None, ["a"])):
        kw = dict(request_ids=ids[:len(args[2])]) if len(args) < 6 else {}
        with pytest.raises(ValueError):
            s.verify(*args, **kw)
        assert (s._shared_draws, dict(s._seeded)) == counters
    assert s.verify(x, drafts, params, q, request_ids=ids) == fresh.verify(x, drafts, params, q, request_ids=ids)
    assert s.sample(x[:2], params, request_ids=ids) == fresh.sample(x[:2], params, request_ids=ids)
