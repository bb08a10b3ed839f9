"""Beam search on an 8-bit output layer with adapters and a paged cache, as a server would run it.

A toy language model: a token's state goes into a cache, the next token follows from the mean of the
row's states and the last one.  Each request has its own adapter on the output layer (or none).
Each step:

    cache of the row -> block_norm (int8) -> int8_linear + adapter_linear (logits)
      -> BeamSearch.step (tokens, parents) -> CachePages.step (the beams' pages) -> the new states

    python examples/beam_step.py [--requests 4] [--beams 4] [--tokens 24]
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "full-inference-engine_amd"))

from fie_amd.adapters import AdapterBank, adapter_linear    # noqa: E402
from fie_amd.beam import BeamSearch                         # noqa: E402
from fie_amd.linear import int8_linear, quantize_rows       # noqa: E402
from fie_amd.norm import block_norm                         # noqa: E402
from fie_amd.pages import CachePages                        # noqa: E402

DEV = "cuda"
PAGE = 8                # tokens of a page


class Toy:
    """Token -> state; a row's states -> logits, the output layer in 8 bits with adapters beside it."""

    def __init__(self, vocab: int, hidden: int, adapters: int, rank: int, seed: int):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
        self.embed = rnd(vocab, hidden).bfloat16()
        self.norm = (1.0 + 0.1 * rnd(hidden)).bfloat16()
        self.weight, self.scale = quantize_rows(6.0 * rnd(vocab, hidden) / hidden ** 0.5)
        self.bank = AdapterBank(adapters, hidden, vocab, rank, torch.bfloat16, DEV)
        for i in range(adapters):
            self.bank.load(i, rnd(rank, hidden) / hidden ** 0.5, rnd(vocab, rank), 1.0)

    def logits(self, last: torch.Tensor, mean: torch.Tensor, plan) -> torch.Tensor:
        got = block_norm(self.embed[last], mean, self.norm, quantize=True)
        base = int8_linear(got.y, self.weight, self.scale, x_scale=got.scale, out_dtype=torch.float32)
        return adapter_linear(got.y, self.bank, plan, x_scale=got.scale, base=base)


def places(pages: CachePages) -> tuple[torch.Tensor, torch.Tensor]:
    """Where each row's tokens are in a cache of [pages * page_size] rows, and which of them are."""
    at = torch.arange(pages.max_pages * PAGE, device=DEV)
    inside = at < pages.lengths[:, None]
    page = pages.table.long().clamp(min=0)[:, at // PAGE]
    return page * PAGE + at % PAGE, inside


def run(requests: int = 4, beams: int = 4, tokens: int = 24, prompt: int = 11, vocab: int = 3000, hidden: int = 256,
        length_penalty: float = 1.0, seed: int = 0) -> dict:
    model = Toy(vocab, hidden, adapters=3, rank=8, seed=seed)
    rows = requests * beams
    most = -(-(prompt + tokens) // PAGE)
    states = torch.zeros(rows * most, PAGE, hidden, dtype=torch.bfloat16, device=DEV)
    ids = torch.zeros(rows * most, PAGE, dtype=torch.int64, device=DEV)
    pages = CachePages(rows * most, PAGE, rows, most, DEV, caches=[states, ids])
    search = BeamSearch(DEV, requests, beams, max_tokens=tokens, eos=[1, 2], length_penalty=length_penalty)
    # whose adapter: requests take turns, every fourth has none
    plan = model.bank.plan(torch.tensor([r % 4 if r % 4 < 3 else -1 for r in range(requests)], dtype=torch.int32,
                                        device=DEV).repeat_interleave(beams))

    def write(row_tokens: torch.Tensor, first: int) -> None:
        """[rows, n] tokens from position ``first`` on."""
        at, _ = places(pages)
        at = at[:, first:first + row_tokens.shape[1]]
        states.view(-1, hidden)[at] = model.embed[row_tokens]
        ids.view(-1)[at] = row_tokens

    # the prompts, in their requests' first rows; the other beams share their pages
    gen = torch.Generator(device=DEV).manual_seed(seed + 1)
    prompts = torch.randint(3, vocab, (requests, prompt), generator=gen, device=DEV).repeat_interleave(beams, 0)
    first = (torch.arange(rows, device=DEV) // beams * beams).int()
    lengths = torch.where(torch.arange(rows, device=DEV) == first, prompt, 0).int()
    if not pages.step(lengths).all():
        raise RuntimeError("the prompts do not fit the pool")
    pages.fork(first)
    write(prompts, 0)
    last, steps = prompts[:, -1], 0
    while steps < tokens and not search.all_done():
        at, inside = places(pages)
        mean = torch.where(inside[:, :, None], states.view(-1, hidden)[at].float(), 0.0).sum(1) / pages.lengths[:, None]
        got = search.step(model.logits(last, mean.bfloat16(), plan))
        if not pages.step(pages.lengths + 1, got.parents).all():
            raise RuntimeError("the pool ran dry")
        last = got.tokens
        write(last[:, None], prompt + steps)
        steps += 1
    pages.compact()
    at, _ = places(pages)
    return dict(answers=[search.answers(r) for r in range(requests)], beams=search.beams, steps=steps, pages=pages,
                prompts=prompts.tolist(), cached=[row[:n] for row, n in zip(ids.view(-1)[at].tolist(), pages.lengths.tolist())])


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--requests", type=int, default=4)
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--tokens", type=int, default=24)
    a = ap.parse_args()
    got = run(a.requests, a.beams, a.tokens)
    print(f"{got['steps']} steps, {got['pages'].pages - got['pages'].free_pages()} pages in use")
    for r, answers in enumerate(got["answers"]):
        print(f"request {r}: {answers[0].value:.3f}", answers[0].tokens[:12], "..")


if __name__ == "__main__":
    main()
