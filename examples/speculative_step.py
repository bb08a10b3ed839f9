"""The end of a decode step on 8-bit weights and drafted tokens, as a server would run it.

A toy language model whose last hidden state is a table lookup stands for the blocks; a cheaper
table drafts.  Each step drafts a few tokens for every request, runs the target on all of them at
once, and keeps what the verification keeps:

    hidden states -> block_norm (residual, norm, int8) -> int8_linear (logits) -> verify

    python examples/speculative_step.py [--requests 8] [--drafts 4] [--steps 16]
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "full-inference-engine_amd"))

from fie_amd import BatchedSampler, SamplingParams          # noqa: E402
from fie_amd.linear import int8_linear, quantize_rows       # noqa: E402
from fie_amd.norm import block_norm                         # noqa: E402

DEV = "cuda"


class Toy:
    """Token -> last block's output and residual -> logits, the output layer in 8 bits."""

    def __init__(self, vocab: int, hidden: int, seed: int):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
        self.block = rnd(vocab, hidden).bfloat16()
        self.embed = rnd(vocab, hidden).bfloat16()
        self.norm = (1.0 + 0.1 * rnd(hidden)).bfloat16()
        self.weight, self.scale = quantize_rows(4.0 * rnd(vocab, hidden) / hidden ** 0.5)

    def hidden(self, tokens: torch.Tensor):
        """The last block's end for these tokens: the int8 input of the output layer."""
        got = block_norm(self.embed[tokens], self.block[tokens], self.norm, quantize=True)
        return got.y, got.scale

    def logits(self, tokens: torch.Tensor) -> torch.Tensor:
        x, x_scale = self.hidden(tokens)
        return int8_linear(x, self.weight, self.scale, x_scale=x_scale, out_dtype=torch.bfloat16)


class Draft:
    """A cheaper model: the target's logits with an error of its own."""

    def __init__(self, target: Toy, noise: float, seed: int):
        self.target, self.noise = target, noise
        self.gen = torch.Generator(device=DEV).manual_seed(seed)

    def probs(self, tokens: torch.Tensor) -> torch.Tensor:
        x = self.target.logits(tokens).float()
        return torch.softmax(x + self.noise * torch.randn(x.shape, generator=self.gen, device=DEV), 1)


def run(requests: int = 8, drafts: int = 4, steps: int = 16, vocab: int = 32000, hidden: int = 1024,
        noise: float = 0.5, seed: int = 0) -> dict:
    target = Toy(vocab, hidden, seed)
    draft = Draft(target, noise, seed + 1)
    params = [SamplingParams(temperature=1.0) if r % 2 else SamplingParams(temperature=0.8, top_p=0.95)
              for r in range(requests)]
    sampler = BatchedSampler(DEV, generator_seed=seed)
    outputs: list[list[int]] = [[r] for r in range(requests)]
    kept = 0
    for _ in range(steps):
        last = torch.tensor([o[-1] for o in outputs], device=DEV)
        # draft: one token a request at a time
        tokens, probs = [last], []
        for _ in range(drafts):
            q = draft.probs(tokens[-1])
            probs.append(q)
            tokens.append(torch.multinomial(q, 1, generator=draft.gen)[:, 0])
        ids = torch.stack(tokens, 1)                                      # [requests, drafts + 1]
        q = torch.stack(probs, 1).view(requests * drafts, vocab)
        # the target's answer after the last token and after each draft, all at once
        logits = target.logits(ids.reshape(-1))
        got = sampler.verify(logits, ids[:, 1:].tolist(), params, q)
        for o, new in zip(outputs, got.token_ids):
            o.extend(new)
        kept += sum(got.accepted)
    new = sum(len(o) - 1 for o in outputs)
    return dict(outputs=outputs, new_tokens=new, kept_share=kept / (requests * drafts * steps),
                tokens_per_step=new / (requests * steps))


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--drafts", type=int, default=4)
    ap.add_argument("--steps", type=int, default=16)
    a = ap.parse_args()
    got = run(a.requests, a.drafts, a.steps)
    print(f"{got['new_tokens']} tokens, {got['tokens_per_step']:.2f} a request and step, "
          f"{100 * got['kept_share']:.0f}% of the drafts kept")
    for o in got["outputs"][:4]:
        print(" ", o[:12], "..")


if __name__ == "__main__":
    main()
