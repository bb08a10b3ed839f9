"""Beams, pages and adapters together on an MI355X: the example, and a search after a verification."""

from __future__ import annotations

import importlib.util
import os

import pytest
import torch

from fie_amd import SamplingParams
from fie_amd.pages import CachePages
from fie_amd.verify import DraftVerifier

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "beam_step.py")
    spec = importlib.util.spec_from_file_location("beam_step", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("requests, beams, tokens, prompt", [(1, 1, 5, 1), (5, 4, 20, 11), (3, 7, 9, 8), (2, 2, 33, 16)])
def test_the_cache_holds_what_the_beams_say(example, requests, beams, tokens, prompt):
    got = example.run(requests=requests, beams=beams, tokens=tokens, prompt=prompt, vocab=500, hidden=64)
    assert 1 <= got["steps"] <= tokens
    for r, answers in enumerate(got["answers"]):
        values = [a.value for a in answers if a.ended]
        assert answers and values == sorted(values, reverse=True)
        assert all(len(a.tokens) <= tokens and all(0 <= t < 500 for t in a.tokens) for a in answers)
        assert all(a.tokens[-1] in (1, 2) or len(a.tokens) == tokens for a in answers if a.ended)
    # rows still searching: prompt and tokens read back through the pages, after they were moved together
    for r in range(requests):
        live = [a for a in got["answers"][r] if not a.ended]
        for b, a in enumerate(live):
            row = got["cached"][r * beams + b]
            assert row[:prompt] == got["prompts"][r * beams] and row[prompt:] == a.tokens
    pages = got["pages"]
    used = pages.pages - pages.free_pages()
    assert used == int(pages.table.max()) + 1 == len(set(pages.table[pages.table >= 0].tolist()))


def test_beams_in_the_middle_of_a_search(example):
    """More tokens than steps taken: every beam is alive, and its cache is its way."""
    got = example.run(requests=4, beams=5, tokens=7, prompt=13, vocab=4000, hidden=64, length_penalty=0.0, seed=3)
    assert got["steps"] == 7 and all(len(a) == 5 for a in got["answers"])
    for r, answers in enumerate(got["answers"]):
        assert {tuple(a.tokens[:-1]) for a in answers if len(a.tokens) == 7} <= {tuple(row[13:-1]) for row in got["cached"][5 * r:5 * r + 5]} | {
            tuple(a.tokens[:-1]) for a in answers if a.tokens[-1] in (1, 2)}


def test_pages_after_a_verification():
    """Refused drafts' pages are free again, kept ones' stay: lengths on the device from the accepted counts."""
    V, lens = 800, [3, 0, 5, 2, 4]
    gen = torch.Generator(device=DEV).manual_seed(1)
    x = 2.0 * torch.randn(sum(lens) + 5, V, generator=gen, device=DEV)
    top = x.argmax(1)
    ids, at = [], 0
    for n in lens:
        ids += [top[at + j] if j < 2 else (top[at + j] + 1) % V for j in range(n)]
        at += n + 1
    v = DraftVerifier(DEV)
    plan = v.plan([SamplingParams()] * 5, lens, V)
    pages = CachePages(40, 2, 5, 12, DEV)
    start = torch.tensor([7, 1, 6, 4, 3], dtype=torch.int32, device=DEV)
    assert pages.step(start).all()
    room = start + torch.tensor(lens, dtype=torch.int32, device=DEV) + 1
    assert pages.step(room).all()
    used = 40 - pages.free_pages()
    got = v.verify(plan, x, torch.stack(ids), torch.rand(len(x), dtype=torch.float64, generator=gen, device=DEV))
    assert got.accepted.tolist() == [2, 0, 2, 2, 2]
    assert pages.step(start + got.accepted + 1).all()
    want = [int(s) + int(a) + 1 for s, a in zip(start, got.accepted)]
    assert pages.lengths.tolist() == want
    assert 40 - pages.free_pages() == sum(-(-n // 2) for n in want) < used
