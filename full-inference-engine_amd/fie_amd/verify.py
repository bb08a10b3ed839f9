"""Verification of drafted tokens on the device (speculative decoding).

A request's drafts are tested, in order, against the distribution the sampler draws from
(temperature, top-k, min-p, top-p, penalties): draft ``d`` with draft probability ``q(d)`` is
kept iff ``u * q(d) < p(d)``; the first refusal is replaced by a draw from what ``p`` has over
``q``, and after the last kept draft the model's next answer is drawn as ``sample`` draws it.
What comes out is distributed as if every token had been sampled one by one, and is at
least one token a request.  Where ``sample`` lets a row's answer depend on its batch (token 0
keeps its penalty only in the widest row), the batch is the rows after as many drafts: those
that one step of ``sample`` would hold.

The reference accepts drafts by argmax only (engine/speculative/acceptance.py); a request
with temperature 0 gives exactly that here.
"""

from __future__ import annotations

import ctypes
from typing import Callable, NamedTuple

import numpy as np
import torch

from . import _lib
from ._lib import VerifyArgs
from .batching.sampler import resolve_params
from .kernel import _DTYPES, FLAG_GREEDY, HELP_ROWS, DeviceStep, FusedSampler
from .runtime.sampling import SamplingParams

FLAG_NO_DRAW = _lib.FIE_FLAG_NO_DRAW
MAX_DRAFTS = _lib.MAX_DRAFTS
_raw_stream = torch._C._cuda_getCurrentRawStream


class Verified(NamedTuple):
    """Device tensors of one verification."""

    tokens: torch.Tensor        # int64 [requests, max_drafts + 1]: kept drafts, one more token, then -1
    accepted: torch.Tensor      # int32 [requests]
    draft_probs: torch.Tensor   # float32 [drafts]: the target's probability of each draft


class VerifyPlan:
    """A batch's settings on the device, for as many steps as they hold: the requests'
    sampling parameters repeated over their rows, and where each request's drafts begin."""

    def __init__(self, fused: FusedSampler, params: list[SamplingParams], draft_lens: list[int], vocab: int,
                 contexts: list[list[int]] | None = None, drafts: list[list[int]] | None = None,
                 rng: np.ndarray | Callable[[VerifyPlan], np.ndarray] | None = None, shared: bool = False):
        # rng as a function is asked for the draws when everything else has been checked, so that
        # a plan that is refused takes none.  shared: the fused sampler's own block of this size,
        # for one call that is waited for
        if len(draft_lens) != len(params):
            raise ValueError("one draft length per request is required")
        lens = np.asarray(draft_lens, dtype=np.int64).reshape(-1)
        if lens.size and (lens.min() < 0 or lens.max() > MAX_DRAFTS):
            raise ValueError(f"draft lengths must be in [0, {MAX_DRAFTS}]")
        if any(p.logprobs is not None for p in params):
            raise ValueError("a verification returns no logprobs")
        if not 1 <= vocab <= _lib.MAX_VOCAB:
            raise ValueError(f"vocab must be in [1, {_lib.MAX_VOCAB}]")
        if (drafts is not None and [len(d) for d in drafts] != lens.tolist()) \
                or (contexts is not None and len(contexts) != len(params)):
            raise ValueError("contexts and drafts must fit the requests and their draft lengths")
        self.requests, self.vocab = len(params), int(vocab)
        self.drafts, self.max_drafts = int(lens.sum()), int(lens.max()) if lens.size else 0
        self.rows = self.drafts + self.requests
        # what a call's tensors have to be
        self.logits_shape, self.probs_shape = (self.rows, self.vocab), (self.drafts, self.vocab)
        self.ids_shape, self.rows_shape = (self.drafts,), (self.rows,)
        row_params = [p for p, n in zip(params, draft_lens) for _ in range(n + 1)]
        row_contexts = None
        if contexts is not None and any(p.has_penalties for p in params):
            if drafts is None:
                raise ValueError("requests with penalties need their drafts on the host")
            row_contexts = [list(c) + list(d[:j]) for c, d in zip(contexts, drafts) for j in range(len(d) + 1)]
        hp = resolve_params(row_params, vocab, None, row_contexts, rng=None if callable(rng) else rng)
        last = np.cumsum(lens + 1) - 1
        no_draw = np.full(self.rows, FLAG_NO_DRAW, dtype=np.int32)
        no_draw[last] = 0
        # last rows without filters: the verification draws from them (the sampler's own kernels
        # do better on the few rows that get span helpers, and on small vocabularies)
        draws = self.rows > HELP_ROWS and vocab > _lib.VERIFY_DRAWS_VOCAB
        if draws:
            plain = ((hp.flags[last] & FLAG_GREEDY) == 0) & (hp.top_k[last] == 0) & (hp.top_p[last] >= 1.0) & (hp.min_p[last] <= 0.0)
            no_draw[last[plain]] = FLAG_NO_DRAW
            draws = bool(plain.any())
        hp.flags = hp.flags | no_draw
        self._offsets = torch.zeros(self.requests + 1, dtype=torch.int64)
        np.cumsum(lens, out=self._offsets.numpy()[1:])
        self._offsets = self._offsets.to(fused.device)
        self.index = self._offsets.get_device()
        self.has_rng = rng is not None
        if callable(rng):
            hp.rng = np.ascontiguousarray(rng(self), dtype=np.uint64).reshape(self.rows, 3)
        # the parameter block, uploaded once
        self._buf = (fused.step_buffers(self.rows, hp.tail_ints()) if shared
                     else DeviceStep(self.rows, hp.tail_ints(), fused.device))
        self._buf.stage(hp)
        self._buf.upload(torch.cuda.current_stream(fused.device))
        a = self._buf.args_of()
        a.rows, a.vocab, a.lp_cols = self.rows, self.vocab, 0
        a.logprobs = a.top_ids = a.top_logprobs = a.chosen_logprob = None
        a.apply_penalties, a.max_row_hist = int(hp.apply_penalties), int(hp.max_row_hist)
        if hp.hist_invalid is not None:
            a.hist_invalid = self._buf.ptr("hist_invalid")
        if hp.rng is not None:
            a.rng = self._buf.ptr("rng")
        self.args = a
        v = VerifyArgs()
        v.requests, v.max_drafts = self.requests, self.max_drafts
        v.draft_offsets, v.draws = self._offsets.data_ptr(), int(draws)
        self.verify_args = v
        self.stream = _raw_stream(self.index)
        self._ready = torch.cuda.Event()
        self._ready.record(torch.cuda.current_stream(fused.device))

    def check(self, logits: torch.Tensor, draft_ids: torch.Tensor, uniforms: torch.Tensor | None,
              draft_probs: torch.Tensor | None) -> None:
        """ValueError where a call's tensors do not fit the plan."""
        rows, drafts, vocab, index = self.rows, self.drafts, self.vocab, self.index
        if logits.shape != self.logits_shape:
            raise ValueError(f"logits must be [{rows}, {vocab}], a request's drafts + 1 rows together")
        if draft_ids.dtype != torch.int64 or draft_ids.shape != self.ids_shape:
            raise ValueError(f"draft_ids must be int64 [{drafts}]")
        if (uniforms is None) != self.has_rng:
            raise ValueError("uniforms are required, or a plan that draws on the device, not both")
        if uniforms is not None and (uniforms.dtype != torch.float64 or uniforms.shape != self.rows_shape):
            raise ValueError(f"uniforms must be float64 [{rows}]")
        if draft_probs is not None and (draft_probs.shape != self.probs_shape or draft_probs.dtype not in _DTYPES):
            raise ValueError(f"draft_probs must be [{drafts}, {vocab}] in float32, float16 or bfloat16")
        for t in (logits, draft_ids, uniforms, draft_probs):
            if t is not None and t.get_device() != index:
                raise ValueError(f"every tensor must be on device {index}")

    def use_on(self, stream: torch.cuda.Stream) -> None:
        """The settings' upload comes before what ``stream`` runs next, and their memory is kept
        for it.  (A stream that captures waits for nothing outside: the upload is then long done.)"""
        if torch.cuda.is_current_stream_capturing():
            return
        stream.wait_event(self._ready)
        for t in (self._buf.dev, self._offsets):
            t.record_stream(stream)


class DraftVerifier:
    """Verifies drafts on one device; calls of one verifier share a workspace and go on one
    stream at a time (going over to another stream, with a wait, is fine: the workspace and the plan's
    memory are kept for both).  A captured call keeps its plan's and the verifier's buffers by address:
    both outlive the graph, plans are made well before the capture, and the largest call (rows,
    vocabulary) goes before it, so that the workspace grows no more."""

    def __init__(self, device: torch.device | str, fused: FusedSampler | None = None):
        self._fused = fused if fused is not None else FusedSampler(device)
        self.device = self._fused.device
        self._run = _lib.launcher("fie_sampler_verify")

    def plan(self, params: list[SamplingParams], draft_lens: list[int], vocab: int,
             contexts: list[list[int]] | None = None, drafts: list[list[int]] | None = None,
             rng: np.ndarray | None = None) -> VerifyPlan:
        """A batch's settings, uploaded once: request i drafts ``draft_lens[i]`` tokens.  With
        penalties, ``contexts`` (the tokens before the drafts) and ``drafts`` are needed.  ``rng``
        (uint64 [rows, 3]) draws on the device, and ``verify`` then takes no uniforms."""
        return VerifyPlan(self._fused, params, draft_lens, vocab, contexts, drafts, rng)

    def verify(self, plan: VerifyPlan, logits: torch.Tensor, draft_ids: torch.Tensor,
               uniforms: torch.Tensor | None = None, draft_probs: torch.Tensor | None = None) -> Verified:
        """One verification on the current stream; nothing waits for it.

        ``logits`` [rows, vocab]: each request's drafts + 1 rows, one request after another;
        row j is the model's answer after j drafts.  ``draft_ids`` int64 [drafts].
        ``uniforms`` float64 [rows] in [0, 1): a row's test of its draft, and on a request's
        last row its draw.  ``draft_probs`` [drafts, vocab]: the distributions the drafts were
        drawn from; without them a draft counts as certain (prompt lookup, argmax drafts)."""
        plan.check(logits, draft_ids, uniforms, draft_probs)
        rows, drafts, vocab, index = plan.rows, plan.drafts, plan.vocab, plan.index
        device = logits.device
        if _raw_stream(index) != plan.stream:
            plan.use_on(torch.cuda.current_stream(index))
        tokens = torch.empty((plan.requests, plan.max_drafts + 1), dtype=torch.int64, device=device)
        accepted = torch.empty(plan.requests, dtype=torch.int32, device=device)
        probs = torch.empty(drafts, dtype=torch.float32, device=device)
        if plan.requests == 0:
            return Verified(tokens, accepted, probs)
        a, v = plan.args, plan.verify_args
        logits, a.dtype = FusedSampler._logits_info(logits)
        draft_ids = draft_ids.contiguous()
        a.logits, a.row_stride = logits.data_ptr(), max(logits.stride(0), vocab)
        if uniforms is not None:
            uniforms = uniforms.contiguous()
            a.uniform = uniforms.data_ptr()
        v.draft_ids = draft_ids.data_ptr() if drafts else None
        v.draft_probs = None
        if draft_probs is not None and drafts:
            draft_probs, v.draft_dtype = FusedSampler._logits_info(draft_probs)
            v.draft_probs, v.draft_stride = draft_probs.data_ptr(), max(draft_probs.stride(0), vocab)
        v.tokens, v.accepted, v.target_probs = tokens.data_ptr(), accepted.data_ptr(), probs.data_ptr()
        ws = self._fused.ensure_workspace(rows, vocab)
        self._run(index, ctypes.byref(a), ctypes.byref(v), ctypes.byref(ws))
        return Verified(tokens, accepted, probs)
