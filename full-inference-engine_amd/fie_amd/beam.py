"""Beam search on the device: the selection over beams and vocabulary, the pool of ended answers,
and the states that go with the beams.

A request's beams are rows next to each other: beam b of request r is row r * beams + b of the
logits and of every state.  ``beam_step`` is one step of all requests; ``reorder_states`` gathers
dense states by the parents it returns, ``fie_amd.pages.CachePages.step`` the pages of a cache.
``BeamSearch`` keeps a batch's beams from step to step and the way back to their tokens.
"""

from __future__ import annotations

import struct
from typing import NamedTuple, Sequence

import numpy as np
import torch

from . import _lib
from ._lib import FIE_BF16, FIE_F16, FIE_F32

_DTYPES = {torch.float32: FIE_F32, torch.float16: FIE_F16, torch.bfloat16: FIE_BF16}
_pack = struct.Struct(_lib.BEAM_ARGS).pack
_run = None             # the library's entry, loaded with the first call
_size = None
_sizes: dict[tuple, int] = {}    # bytes of workspace by a call's device, type and sizes
_F32, _I32 = torch.float32, torch.int32
_INF = float("inf")
_reorder = None
_raw_stream = torch._C._cuda_getCurrentRawStream
MAX_STATES = 48         # tensors of one launch
_packs: dict[int, object] = {}
MAX_BEAMS = 64
MAX_EOS = 16
_NO_EOS = (0,) * MAX_EOS
MAX_ROWS = 65535


class Beams(NamedTuple):
    """The beams of some requests between two steps, on the device."""

    scores: torch.Tensor        # float32 [requests, beams] sums of log-probabilities; -inf: no such beam
    lengths: torch.Tensor       # int32 [requests] tokens chosen so far
    done: torch.Tensor          # bool [requests]
    pool: torch.Tensor          # float32 [requests, beams] ended answers' values, the best first; -inf: none
    ends: torch.Tensor          # int32 [requests, beams, 3] theirs: length, parent row, eos token


class BeamStep(NamedTuple):
    beams: Beams
    tokens: torch.Tensor        # int64 [rows] the token each row goes on with
    parents: torch.Tensor       # int32 [rows] the row that it went on from


def first_beams(requests: int, beams: int, device: torch.device | str) -> Beams:
    """Before the first step: a request's first row is its only beam."""
    scores = torch.full((requests, beams), -_INF, dtype=_F32, device=device)
    scores[:, :1] = 0.0
    return Beams(scores, torch.zeros(requests, dtype=torch.int32, device=device),
                 torch.zeros(requests, dtype=torch.bool, device=device),
                 torch.full((requests, beams), -_INF, dtype=_F32, device=device),
                 torch.full((requests, beams, 3), -1, dtype=torch.int32, device=device))


def beam_step(logits: torch.Tensor, beams: Beams, *, eos: Sequence[int] = (), length_penalty: float = 1.0,
              early_stopping: bool = False, min_tokens: int = 0, max_tokens: int = 0, pad: int = 0, inplace: bool = False,
              history: tuple[torch.Tensor, torch.Tensor] | None = None) -> BeamStep:
    """One step of beam search: ``logits`` [requests * beams, vocab] (float32, float16, bfloat16).

    A continuation's score is its beam's and the token's log-probability, added in 64 bits and
    rounded once (a row's sum of exponentials alone has terms in fp32: its logarithm is off by about
    1e-7).  Continuations rank by their totals, then lower beam, larger logit, lower token.  The
    best ``beams`` of a request that are not in ``eos`` go on.  An ending one among its best
    ``beams`` of all joins the request's pool at total / (length + 1) ** ``length_penalty``; before
    ``min_tokens`` tokens none exists, and with ``max_tokens`` those of that many tokens all end.
    A request is done when its pool is full and, unless ``early_stopping``, the best that goes on
    is no better than the pool's worst; or when nothing goes on.  Rows of a request that is done,
    and rows beside its last beam, come out with score -inf, token ``pad`` and themselves as parent,
    and their logits are not read at the next step.

    A NaN logit counts as -inf, +inf as the largest float32; tokens masked with -inf do not exist.
    Scores and values below the least float32 are held at it.
    ``inplace`` writes the new beams over the old.  ``history``: int32 [steps, rows] tokens and
    parents; a step's are kept at its request's length.  Runs on the current stream; nothing waits
    for it."""
    scores, lengths, done, pool, ends = beams
    if scores.ndim != 2:
        raise ValueError("scores must be [requests, beams]")
    requests, count = shape = scores.shape
    rows = requests * count
    if not 1 <= count <= MAX_BEAMS or rows > MAX_ROWS:
        raise ValueError(f"beams must be in [1, {MAX_BEAMS}], rows at most {MAX_ROWS}")
    index = scores.get_device()
    if index < 0:
        raise ValueError("beam_step runs on a HIP device")
    if not (scores.dtype == pool.dtype == _F32 and lengths.dtype == ends.dtype == _I32 and done.dtype == torch.bool
            and pool.shape == shape and lengths.shape == done.shape == (requests,) and ends.shape == (requests, count, 3)
            and scores.is_contiguous() and lengths.is_contiguous() and done.is_contiguous() and pool.is_contiguous()
            and ends.is_contiguous()):
        raise ValueError(f"beams must be contiguous float32 scores and pool [{requests}, {count}], int32 lengths [{requests}], "
                         f"bool done [{requests}] and int32 ends [{requests}, {count}, 3]")
    if logits.ndim != 2 or logits.shape[0] != rows:
        raise ValueError(f"logits must be [{rows}, vocab], a request's beams together")
    vocab = logits.shape[1]
    code = _DTYPES.get(logits.dtype)
    if code is None:
        raise ValueError("logits must be float32, float16 or bfloat16")
    if not 1 <= vocab <= _lib.MAX_VOCAB:
        raise ValueError(f"vocab must be in [1, {_lib.MAX_VOCAB}]")
    if not (index == logits.get_device() == lengths.get_device() == done.get_device() == pool.get_device() == ends.get_device()):
        raise ValueError("every tensor must be on the scores' device")
    stop = len(eos)
    if stop > MAX_EOS or (stop and not 0 <= min(eos) <= max(eos) < vocab):
        raise ValueError(f"eos: at most {MAX_EOS} tokens of the vocabulary")
    if not -_INF < length_penalty < _INF or not 0 <= pad < 1 << 31 or not 0 <= min_tokens < 1 << 31 \
            or not 0 <= max_tokens < 1 << 31:
        raise ValueError("length_penalty must be a finite number, pad, min_tokens and max_tokens whole numbers of 31 bits")
    h_tokens = h_parents = h_steps = 0
    if history is not None:
        for t in history:
            if t.dtype != _I32 or t.ndim != 2 or t.shape[1] != rows or t.shape != history[0].shape \
                    or not t.is_contiguous() or t.get_device() != index:
                raise ValueError(f"history must be two contiguous int32 [steps, {rows}] on the scores' device")
        h_tokens, h_parents, h_steps = history[0].data_ptr(), history[1].data_ptr(), history[0].shape[0]
    stride, step = logits.stride()
    if (vocab > 1 and step != 1) or (rows > 1 and stride < vocab):
        logits, stride = logits.contiguous(), vocab
    like = torch.empty_like
    new = beams if inplace else Beams(like(scores), like(lengths), like(done), like(pool), like(ends))
    tokens = scores.new_empty(rows, dtype=torch.int64)
    parents = lengths.new_empty(rows)
    if rows:
        global _run, _size
        if _run is None:
            _run, _size = _lib.launcher("fie_beam_step"), _lib.load().fie_beam_workspace_size
        args = [logits.data_ptr(), scores.data_ptr(), lengths.data_ptr(), done.data_ptr(), pool.data_ptr(), ends.data_ptr(),
                new.scores.data_ptr(), new.lengths.data_ptr(), new.done.data_ptr(), new.pool.data_ptr(), new.ends.data_ptr(),
                tokens.data_ptr(), parents.data_ptr(), h_tokens, h_parents, max(stride, vocab), 0, 0, length_penalty, requests,
                count, vocab, code, early_stopping, min_tokens, pad, h_steps, stop, *eos, *_NO_EOS[stop:], max_tokens]
        key = index, code, requests, count, vocab, stop
        size = _sizes.get(key)
        if size is None:
            if len(_sizes) > 256:
                _sizes.clear()
            size = _sizes[key] = _size(_pack(*args))
        room = done.new_empty(size)
        args[16], args[17] = room.data_ptr(), size
        _run(index, _pack(*args))
    return BeamStep(new, tokens, parents)


def reorder_states(states: Sequence[torch.Tensor], parents: torch.Tensor,
                   out: Sequence[torch.Tensor] | None = None) -> list[torch.Tensor]:
    """``[s[parents] for s in states]`` in one launch: states [rows, ...] of any types, ``parents`` int32
    [n] rows (one outside [0, rows) stands for the row's own number, which has to be one of the
    states').  ``out``: as many tensors [n, ...] to write into, apart from all states and from each
    other.  Runs on the current stream; nothing waits for it."""
    if parents.dtype != torch.int32 or parents.ndim != 1:
        raise ValueError("parents must be int32 [rows]")
    index = parents.get_device()
    if index < 0:
        raise ValueError("reorder_states runs on a HIP device")
    n = parents.shape[0]
    if not parents.is_contiguous():
        parents = parents.contiguous()
    if out is not None and len(out) != len(states):
        raise ValueError("as many outputs as states")
    got, flat, held = [], [], []                    # held: copies, until the launch
    for i, s in enumerate(states):
        if s.ndim < 1 or s.get_device() != index:
            raise ValueError("states must be [rows, ...] on the parents' device")
        shape = s.shape
        rows = shape[0]
        if n > rows:
            raise ValueError(f"{n} parents of {rows} rows")
        if s.is_conj() or s.is_neg():               # another's memory, to be read as such
            s = s.resolve_conj().resolve_neg()
            held.append(s)
        dense = s.is_contiguous()
        if not dense and rows and not s[0].is_contiguous():
            s, dense = s.contiguous(), True
            held.append(s)
        if out is None:
            t = torch.empty_like(s) if dense and n == rows else s.new_empty((n, *shape[1:]))
        else:
            t = out[i]
            if t.dtype != s.dtype or t.shape != (n, *shape[1:]) or t.get_device() != index or t.is_conj() or t.is_neg():
                raise ValueError(f"output {i} must be [{n}, ...] as its state")
            if not t.is_contiguous() and n and (not t[0].is_contiguous() or (n > 1 and t.numel() and t.stride(0) < t[0].numel())):
                raise ValueError("outputs need contiguous rows that do not overlap")
        got.append(t)
        width = s.numel()
        if width and n:
            size = s.element_size()
            width = width // rows * size
            flat += (s.data_ptr(), t.data_ptr(), width if dense else s.stride(0) * size,
                     width if out is None else t.stride(0) * size, width, rows)
    if out is not None and flat and _cross(flat, n, parents.data_ptr()):
        raise ValueError("an output overlaps a state, the parents or another output")
    global _reorder
    if flat and _reorder is None:
        _reorder = _lib.launcher("fie_reorder_states")
    for at in range(0, len(flat), 6 * MAX_STATES):
        some = flat[at:at + 6 * MAX_STATES]
        count = len(some) // 6
        pack = _packs.get(count)
        if pack is None:
            pack = _packs[count] = struct.Struct(_lib.STATES_ARGS + _lib.STATE_ARGS * count).pack
        _reorder(index, pack(parents.data_ptr(), n, count, *some))
    return got


def _cross(flat: list, n: int, parents: int) -> bool:
    """Whether an output (of n rows) has memory of a state's, another output's or the parents': ``flat`` has (state, output, their
    strides, width, rows of the state) in bytes.  Rows of one stride may lie between each other's."""
    # first byte and end, stride (0: one piece), width, an output
    parts = [(parents, parents + 4 * n, 0, 4 * n, False)]
    for i in range(0, len(flat), 6):
        s, t, s_stride, t_stride, width, rows = flat[i:i + 6]
        parts.append((s, s + (rows - 1) * s_stride + width, s_stride if rows > 1 else 0, width, False))
        parts.append((t, t + (n - 1) * t_stride + width, t_stride if n > 1 else 0, width, True))
    parts.sort()
    some: list = []                                 # that meet in a chain
    end = 0
    for p in parts:
        if p[0] >= end:                             # apart from all before it
            if len(some) > 1 and _meet(some):
                return True
            some = []
        some.append(p)
        end = max(end, p[1])
    return len(some) > 1 and _meet(some)


def _meet(parts: list) -> bool:
    stride = max(p[2] for p in parts)
    if stride and len(parts) > 8 and all(p[2] == stride for p in parts):
        # columns of one buffer: two rounds of their places in a row
        at = sorted((p[0] % stride, p[3], p[4]) for p in parts)
        every = outs = 0
        for first, width, out in at + [(first + stride, width, out) for first, width, out in at]:
            if first < (every if out else outs):
                break
            every = max(every, first + width)
            outs = max(outs, first + width) if out else outs
        else:
            return False
    return any(_shared(q, p) for i, p in enumerate(parts) for q in parts[:i] if p[4] or q[4])


def _shared(a: tuple, b: tuple) -> bool:
    """Whether rows of (first byte, end, stride or 0 for one piece, width) have memory in common."""
    if a[1] <= b[0] or b[1] <= a[0]:
        return False
    if a[2] and b[2] and a[2] != b[2]:
        return True                                 # (rows of two strides that miss each other are not looked for)
    stride = a[2] or b[2]
    at = (b[0] - a[0]) % stride if stride else 0
    return at < a[3] or stride - at < b[3]


class Answer(NamedTuple):
    value: float                # score / length ** length_penalty
    tokens: list[int]           # its eos among them, if it ended with one
    ended: bool


class BeamSearch:
    """The beams of up to ``requests`` requests from step to step on one device; ``step`` takes a model's
    logits and says which token each row goes on with and which row it went on from.

        search = BeamSearch(device, requests, beams, max_tokens=200, eos=[2])
        while not search.all_done():                     # or so many steps: nothing else waits
            got = search.step(model(tokens, caches))
            pages.step(pages.lengths + 1, got.parents)   # fie_amd.pages: the beams' caches
            tokens = got.tokens
        best = search.answers(0)[0]

    A request's slot is used again after ``restart``.  Calls of one search go on one stream at a
    time."""

    def __init__(self, device: torch.device | str, requests: int, beams: int, *, max_tokens: int,
                 eos: Sequence[int] = (), length_penalty: float = 1.0, early_stopping: bool = False, min_tokens: int = 0,
                 pad: int = 0):
        if requests < 1 or not 1 <= beams <= MAX_BEAMS or requests * beams > MAX_ROWS:
            raise ValueError(f"beams must be in [1, {MAX_BEAMS}], rows in [1, {MAX_ROWS}]")
        if max_tokens < 1:
            raise ValueError("max_tokens must be at least 1")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError("BeamSearch runs on a HIP device")
        self.requests, self.count, self.max_tokens = requests, beams, max_tokens
        self._settings = dict(eos=tuple(eos), length_penalty=length_penalty, early_stopping=early_stopping,
                              min_tokens=min_tokens, max_tokens=max_tokens, pad=pad)
        self.beams = first_beams(requests, beams, self.device)
        rows = requests * beams
        self._history = (torch.zeros((max_tokens, rows), dtype=torch.int32, device=self.device),
                         torch.zeros((max_tokens, rows), dtype=torch.int32, device=self.device))
        self.device, self._index = self.beams.scores.device, self.beams.scores.get_device()
        self._made_on = _raw_stream(self._index)

    def _on_stream(self) -> None:
        """Memory made on another stream is kept for this one."""
        if _raw_stream(self._index) != self._made_on and not torch.cuda.is_current_stream_capturing():
            stream = torch.cuda.current_stream(self._index)
            for t in (*self.beams, *self._history):
                t.record_stream(stream)

    def step(self, logits: torch.Tensor) -> BeamStep:
        """One step of every request (``beam_step``); the beams are written over."""
        self._on_stream()
        return beam_step(logits, self.beams, inplace=True, history=self._history, **self._settings)

    def _slots(self, requests: Sequence[int]) -> torch.Tensor:
        if any(not 0 <= r < self.requests for r in requests):
            raise ValueError(f"requests must be in [0, {self.requests})")
        return torch.tensor(list(requests), dtype=torch.int64).to(self.device)

    def restart(self, requests: Sequence[int]) -> None:
        """These requests' slots begin anew."""
        at = self._slots(requests)
        self._on_stream()
        for t, fresh in zip(self.beams, first_beams(len(requests), self.count, self.device)):
            t[at] = fresh

    def stop(self, requests: Sequence[int]) -> None:
        """These requests are done as they are, or were never begun (slots that only fill up the batch): their
        logits are not read until ``restart``.  Beams that had not ended are dropped."""
        at = self._slots(requests)
        self._on_stream()
        self.beams.done[at] = True

    def all_done(self) -> bool:
        """Whether every request is done (waits for the device)."""
        return bool(self.beams.done.all())

    def answers(self, request: int) -> list[Answer]:
        """A request's ended answers, the best first, and while it is not done its beams behind them
        (waits for the device)."""
        if not 0 <= request < self.requests:
            raise ValueError(f"request must be in [0, {self.requests})")
        scores, length, done, pool, ends = (t[request].cpu().numpy() for t in self.beams)
        rows = slice(request * self.count, (request + 1) * self.count)
        steps = min(int(length), self.max_tokens)
        tokens, parents = (t[:steps, rows].cpu().numpy() for t in self._history)

        def way(row: int, n: int) -> list[int]:
            got = []
            for t in range(n - 1, -1, -1):
                got.append(int(tokens[t, row]))
                row = int(parents[t, row]) - rows.start
            return got[::-1]

        got = [Answer(float(v), way(int(p) - rows.start, int(n) - 1) + [int(t)], True)
               for v, (n, p, t) in zip(pool, ends) if v > -np.inf]
        if not done and length:
            with np.errstate(all="ignore"):             # (as the kernel: a power out of range is 0 or an infinity)
                scale = np.float64(length) ** self._settings["length_penalty"]
                values = np.where(scores != 0.0, np.maximum(scores / scale, np.finfo(np.float32).min), 0.0)
            got += [Answer(float(v), way(b, steps), False) for b, (s, v) in enumerate(zip(scores, values)) if s > -np.inf]
        return got
