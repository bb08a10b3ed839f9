"""Pages of a cache: tables, lengths and counts of holders on the device, and what moves them.

A pool of ``pages`` pages of ``page_size`` tokens serves ``rows`` sequences, each with a table of
its pages.  Rows may share pages: a beam those of the beam it went on from, a sequence its
prefix's.  One call makes the step of a batch:

    fork      a row takes the pages of its parent (``parents``)
    cut       a row keeps as many tokens as ``lengths`` says; pages that no row holds are free
    grow      a row gets the pages for more tokens, and a last page of its own to write into: one
              that is not full and that others hold is copied

``compact`` moves the used pages together to the lowest numbers.  Which page goes where is settled
by the rows' order and the pages' numbers alone, so a call gives the same tables every time.
"""

from __future__ import annotations

import struct
from typing import Sequence

import torch

from . import _lib

_pack = struct.Struct(_lib.PAGES_ARGS + _lib.GROUP_ARGS * 8).pack
_runs: dict[str, object] = {}           # the library's entries, loaded with the first call
_raw_stream = torch._C._cuda_getCurrentRawStream
MAX_ROWS = 4096
MAX_PAGES = 1 << 21
MAX_GROUPS = 8


def _launch(name: str, index: int, args: bytes) -> None:
    run = _runs.get(name)
    if run is None:
        run = _runs[name] = _lib.launcher(name)
    run(index, args)


class CachePages:
    """The pages of ``rows`` sequences on one device, and the cache tensors that they are pages of.

    ``state`` (int32) is everything that calls change, ``table`` [rows, max_pages] (-1 past a row's
    pages), ``lengths`` [rows] and ``refs`` [pages] (rows that hold a page) views of it; a copy of it
    put back later undoes what was done to the tables in between, though not what was written into
    pages.  Calls go on the current stream, one stream at a time, and wait for nothing; one that is
    captured keeps the object's buffers by address, and the object outlives the graph."""

    def __init__(self, pages: int, page_size: int, rows: int, max_pages: int, device: torch.device | str, *,
                 caches: Sequence[torch.Tensor] = (), token_dim: int | None = 1):
        if not 1 <= pages <= MAX_PAGES or not 1 <= page_size <= 65536:
            raise ValueError(f"pages must be in [1, {MAX_PAGES}], page_size in [1, 65536]")
        if not 1 <= rows <= MAX_ROWS or not 1 <= max_pages <= pages:
            raise ValueError(f"rows must be in [1, {MAX_ROWS}], max_pages in [1, pages]")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError("CachePages runs on a HIP device")
        lib = _lib.load()
        self.pages, self.page_size, self.rows, self.max_pages = pages, page_size, rows, max_pages
        self.state = torch.zeros(lib.fie_pages_state_ints(pages, rows, max_pages), dtype=torch.int32, device=self.device)
        self.device, self._index = self.state.device, self.state.get_device()
        self.table, self.lengths, self.refs, self._blocks = self._parts(self.state)
        self._scratch = torch.empty(lib.fie_pages_scratch_bytes(pages, rows), dtype=torch.uint8, device=self.device)
        self._made_on = _raw_stream(self._index)
        self._groups: list[tuple] = []          # (layout, tensors, their addresses on the device)
        self.table.fill_(-1)
        self._count_blocks()
        if len(caches):
            self.add_caches(caches, token_dim)

    def _parts(self, state: torch.Tensor) -> tuple[torch.Tensor, ...]:
        n = self.rows * self.max_pages
        return (state[:n].view(self.rows, self.max_pages), state[n:n + self.rows],
                state[n + self.rows:n + self.rows + self.pages], state[n + self.rows + self.pages:])

    def _count_blocks(self) -> None:
        free = torch.nn.functional.pad((self.refs == 0).int(), (0, -self.pages % 1024))
        self._blocks.copy_(free.view(-1, 1024).sum(1))

    # ------------------------------------------------------------------ the caches
    def add_caches(self, caches: Sequence[torch.Tensor], token_dim: int | None = 1) -> None:
        """Tensors [pages, ...] that go along when pages are copied.  ``token_dim`` is the dimension of a page's
        tokens, everything past it contiguous: 1 for [pages, page_size, heads, dim], 2 for [pages, heads,
        page_size, dim]; None where a page has values for all its tokens together (scales).  Pages may lie
        between each other ([heads, pages, page_size, dim], transposed)."""
        groups: dict[tuple, list[torch.Tensor]] = {}
        for t in caches:
            if t.get_device() != self._index:
                raise ValueError("caches must be on the pages' device")
            at = t.ndim if token_dim is None else token_dim
            if t.ndim < 1 or t.shape[0] != self.pages or not 1 <= at <= t.ndim or (
                    token_dim is not None and (at == t.ndim or t.shape[at] != self.page_size)):
                raise ValueError(f"a cache must be [{self.pages}, ...] with {self.page_size} tokens in dimension token_dim")
            if t.numel() == 0:
                continue
            size = t.element_size()
            inner = 1                           # elements that lie together: behind the tokens, or a whole page's
            if token_dim is None:
                if not t[0].is_contiguous():
                    raise ValueError("a cache without tokens needs contiguous pages")
                outer, outer_stride, token = 1, 0, t[0].numel() * size
            else:
                if not _dense(t, at):
                    raise ValueError("a cache must be contiguous from its tokens on")
                for n in t.shape[at + 1:]:
                    inner *= n
                outer, outer_stride, token = *_pieces(t, at), inner * size
            piece, step, pitch = token * (1 if token_dim is None else self.page_size), t.stride(0) * size, outer_stride * size
            # a page's pieces lie together, or all pages' first pieces do, then all second ones
            if self.pages > 1 and step < (outer - 1) * pitch + piece \
                    and not (step >= piece and pitch >= (self.pages - 1) * step + piece):
                raise ValueError("a cache's pages overlap")
            key = (step, pitch, token, outer, int(token_dim is None))
            groups.setdefault(key, []).append(t)
        if len(self._groups) + len(groups) > MAX_GROUPS:
            raise ValueError(f"caches of more than {MAX_GROUPS} layouts")
        for (stride, outer_stride, token, outer, whole), tensors in groups.items():
            base = torch.tensor([t.data_ptr() for t in tensors], dtype=torch.int64).to(self.device)
            shift = int(any(v % 16 for v in (stride, outer_stride, *(t.data_ptr() for t in tensors))))
            self._groups.append(((stride, outer_stride, token, len(tensors), outer, whole, shift), tensors, base))
        self._mixed |= bool(groups) and _raw_stream(self._index) != self._made_on
        self._packed = None

    _packed: list | None = None
    _mixed = False                      # addresses of caches made on another stream than the state

    def _args(self, parents: int, lengths: int, granted: int, live: int, src: int, dst: int, copies: int) -> bytes:
        p = self._packed
        if p is None:
            flat = [v for layout, _, base in self._groups for v in (base.data_ptr(), *layout)]
            p = self._packed = flat + [0] * (8 * (MAX_GROUPS - len(self._groups)))
        return _pack(self.state.data_ptr(), self._scratch.data_ptr(), self._scratch.numel(), self.pages, self.page_size, self.rows,
                     self.max_pages, parents, lengths, granted, live, src, dst, copies, len(self._groups), *p)

    def _on_stream(self) -> None:
        """Memory made on another stream is kept for this one."""
        if (self._mixed or _raw_stream(self._index) != self._made_on) and not torch.cuda.is_current_stream_capturing():
            stream = torch.cuda.current_stream(self._index)
            for t in (self.state, self._scratch, *(base for _, _, base in self._groups)):
                t.record_stream(stream)

    # ------------------------------------------------------------------ the calls
    def _vector(self, t: torch.Tensor, name: str, size: int) -> torch.Tensor:
        if t.dtype != torch.int32 or t.shape != (size,) or t.get_device() != self._index:
            raise ValueError(f"{name} must be int32 [{size}] on the pages' device")
        return t.contiguous()

    def step(self, lengths: torch.Tensor | None, parents: torch.Tensor | None = None) -> torch.Tensor:
        """Rows fork from ``parents`` and have ``lengths`` tokens afterwards; returns which got them (bool [rows]).

        ``parents`` int32 [rows]: row i takes the pages and tokens of row parents[i] (None: its own;
        outside [0, rows): it is emptied).  ``lengths`` int32 [rows]: fewer tokens than its parent's
        cut the row (0 frees it), more grow it (None: its parent's).  Rows get pages in their order,
        the lowest free ones; a row whose pages, with those of the rows before it, are more than are
        free, or more than ``max_pages``, keeps its parent's tokens, cut as asked, and does not grow.

        A row that grows from a last page that is not full and that other rows hold gets a copy of
        its tokens there; where all holders grow, the longest of them, and of those the lowest row,
        keeps it.  So what a row writes past its old tokens is its own."""
        p = self._vector(parents, "parents", self.rows) if parents is not None else None
        n = self._vector(lengths, "lengths", self.rows) if lengths is not None else None
        granted = torch.empty(self.rows, dtype=torch.bool, device=self.device)
        self._on_stream()
        _launch("fie_pages_step", self._index, self._args(p.data_ptr() if p is not None else 0, n.data_ptr() if n is not None else 0,
                                                          granted.data_ptr(), 0, 0, 0, 0))
        return granted

    def fork(self, parents: torch.Tensor) -> None:
        """Row i takes the pages of row parents[i] (``step`` without lengths)."""
        self.step(None, parents)

    def compact(self) -> torch.Tensor:
        """The used pages move to the numbers below their count, in order; returns the count (int32).
        Numbers of pages kept outside the table mean nothing afterwards."""
        live = torch.empty((), dtype=torch.int32, device=self.device)
        self._on_stream()
        _launch("fie_pages_compact", self._index, self._args(0, 0, 0, live.data_ptr(), 0, 0, 0))
        return live

    def copy_pages(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Pages dst[i] of the caches become copies of src[i] (int32; a pair with a number that is no page is
        left out).  No page is both source and destination, or a destination twice."""
        n = src.numel()
        src, dst = self._vector(src, "src", n), self._vector(dst, "dst", n)
        if not n:
            return
        self._on_stream()
        _launch("fie_pages_copy", self._index, self._args(0, 0, 0, 0, src.data_ptr(), dst.data_ptr(), n))

    def free_pages(self) -> int:
        """How many pages no row holds (waits for the device)."""
        return int(self._blocks.sum())

    def load(self, table: torch.Tensor, lengths: torch.Tensor) -> None:
        """Begins with these rows' pages (waits for the device).  Entries past a row's pages are taken as -1;
        rows that share a page have it at the same place."""
        # 64 bits: a cut to 32 could make a page or a length of what is none
        table, lengths = (t.to(self.device, torch.float64 if t.is_floating_point() else torch.int64) for t in (table, lengths))
        if table.shape != self.table.shape or lengths.shape != self.lengths.shape:
            raise ValueError(f"table must be [{self.rows}, {self.max_pages}], lengths [{self.rows}]")
        most = min(self.max_pages * self.page_size, (1 << 31) - 1)
        if not bool(((lengths >= 0) & (lengths <= most)).all()):
            raise ValueError("lengths must be in [0, max_pages * page_size], 31 bits at most")
        col = torch.arange(self.max_pages, device=self.device)
        used = col < ((lengths.long() + self.page_size - 1) // self.page_size)[:, None]
        ids = table[used]
        if ids.numel() and (int(ids.min()) < 0 or int(ids.max()) >= self.pages):
            raise ValueError(f"a row's pages must be in [0, {self.pages})")
        ids = ids.long()
        at = col.expand_as(table)[used]
        place = torch.full((self.pages,), -1, dtype=torch.int64, device=self.device).scatter_reduce_(0, ids, at, "amax")
        if bool((place[ids] != at).any()):
            raise ValueError("a page is at two places")
        self._on_stream()
        self.table.copy_(torch.where(used, table, -1))
        self.lengths.copy_(lengths)
        self.refs.copy_(torch.bincount(ids, minlength=self.pages))
        self._count_blocks()


def _dense(t: torch.Tensor, at: int) -> bool:
    """Whether the dimensions from ``at`` on lie together."""
    step = 1
    for n, stride in zip(reversed(t.shape[at:]), reversed(t.stride()[at:])):
        if n > 1 and stride != step:
            return False
        step *= n
    return True


def _pieces(t: torch.Tensor, at: int) -> tuple[int, int]:
    """The dimensions between the pages and ``at`` as one: how many, and the elements between them."""
    count, stride = 1, 0
    for n, s in zip(reversed(t.shape[1:at]), reversed(t.stride()[1:at])):
        if n == 1:
            continue
        if count > 1 and s != count * stride:
            raise ValueError("a cache's dimensions in front of its tokens must lie together")
        if count == 1:
            stride = s
        count *= n
    return count, stride
