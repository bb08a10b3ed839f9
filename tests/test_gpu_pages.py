"""Pages of a cache on an MI355X against a plain account of them: every number and byte is equal."""

from __future__ import annotations

import random

import numpy as np
import pytest
import torch

from fie_amd.pages import CachePages

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Plain:
    """Rows' pages and the caches' tokens, row by row."""

    def __init__(self, pages, page, rows, wide, caches=()):
        self.n, self.page, self.rows, self.wide = pages, page, rows, wide
        self.table, self.lengths = [[] for _ in range(rows)], [0] * rows
        self.caches = [c.clone() for c in caches]       # [pages, page, ...]

    def refs(self):
        got = [0] * self.n
        for row in self.table:
            for p in row:
                got[p] += 1
        return got

    def up(self, tokens):
        return -(-tokens // self.page)

    def step(self, lengths, parents=None):
        parents = list(range(self.rows)) if parents is None else parents
        old, have = self.table, self.lengths
        held, table = [], []
        for i, p in enumerate(parents):
            if not 0 <= p < self.rows:
                held.append(0)
                table.append([])
                continue
            n = have[p] if lengths is None else max(0, min(lengths[i], have[p]))
            held.append(n)
            table.append(list(old[p][:self.up(n)]))
        self.table, self.lengths = table, list(held)
        want = held if lengths is None else [max(a, b) for a, b in zip(lengths, held)]
        refs, writers = self.refs(), {}
        fits = [self.up(w) <= self.wide for w in want]
        for i in range(self.rows):
            if want[i] > held[i] and fits[i] and held[i] % self.page:
                writers.setdefault(table[i][-1], []).append((-(held[i] % self.page), i))
        free = iter([p for p in range(self.n) if refs[p] == 0])
        left = refs.count(0)
        granted, copies = [], []
        for i in range(self.rows):
            if want[i] <= held[i] or not fits[i]:
                granted.append(want[i] <= held[i])
                continue
            copy = False
            if held[i] % self.page:
                mine = writers[table[i][-1]]
                copy = not (len(mine) == refs[table[i][-1]] and min(mine)[1] == i)
            need = self.up(want[i]) - self.up(held[i]) + copy
            left -= need                                # rows behind one without pages have to need none
            if need and left < 0:
                granted.append(False)
                continue
            granted.append(True)
            if copy:
                copies.append((table[i][-1], next(free), held[i] % self.page))
                table[i][-1] = copies[-1][1]
            table[i] += [next(free) for _ in range(self.up(want[i]) - len(table[i]))]
            self.lengths[i] = want[i]
        for src, dst, fill in copies:
            for c in self.caches:
                c[dst, :fill] = c[src, :fill]
        return granted

    def compact(self):
        refs = self.refs()
        used = sum(r > 0 for r in refs)
        to = dict(zip([p for p in range(used, self.n) if refs[p]], [p for p in range(used) if not refs[p]]))
        for src, dst in to.items():
            for c in self.caches:
                c[dst] = c[src]
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        return used


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def same(pool, plain, caches=None):
    torch.cuda.synchronize()
    table = np.full((plain.rows, plain.wide), -1)
    for i, row in enumerate(plain.table):
        table[i, :len(row)] = row
    np.testing.assert_array_equal(pool.table.cpu().numpy(), table)
    assert pool.lengths.tolist() == plain.lengths
    refs = plain.refs()
    assert pool.refs.tolist() == refs
    free = np.zeros(-(-plain.n // 1024) * 1024, int)
    free[:plain.n] = np.array(refs) == 0
    np.testing.assert_array_equal(pool._blocks.cpu().numpy(), free.reshape(-1, 1024).sum(1))
    for c, d in zip(caches or (), plain.caches):
        assert torch.equal(c, d)


def caches(pages, page, kinds=("bf16",), seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    make = dict(bf16=lambda: rnd(pages, page, 2, 24).bfloat16(), fp32=lambda: rnd(pages, page, 3),
                odd=lambda: torch.randint(0, 255, (pages, page, 7), generator=gen, device=DEV, dtype=torch.uint8))
    return [make[k]() for k in kinds]


@pytest.mark.parametrize("pages, page, rows, wide", [(1, 1, 1, 1), (7, 3, 2, 5), (40, 4, 6, 9), (100, 16, 12, 20), (1024, 8, 33, 40),
                                                     (1025, 1, 64, 60), (3000, 2, 130, 25), (5000, 5, 1100, 12)])
def test_any_course_of_steps(pages, page, rows, wide):
    """Random forks, cuts and growths, pools that run dry, and now and then all of it moved together."""
    print(f"  case: {pages} x {page}, {rows} x {wide}", flush=True)
    rng = random.Random(pages)
    mine = caches(pages, page, ("bf16", "odd", "fp32"))
    pool, plain = CachePages(pages, page, rows, wide, DEV, caches=mine), Plain(pages, page, rows, wide, mine)
    same(pool, plain)
    for t in range(12 if rows > 500 else 30):
        parents = None
        if rng.random() < 0.6:
            parents = [rng.randrange(rows) if rng.random() < 0.5 else i for i in range(rows)]
            for _ in range(rng.randrange(3)):
                parents[rng.randrange(rows)] = rng.choice((-1, rows, -2 ** 31, 2 ** 31 - 1))
        lengths = None
        if rng.random() < 0.9:
            at = [plain.lengths[p] if 0 <= p < rows else 0 for p in (parents or range(rows))]
            kind = rng.choice(("one", "few", "any", "over"))
            most = wide * page + (5 if kind == "over" else 0)
            lengths = [{"one": n + 1, "few": max(0, n + rng.randint(-2 * page, 2 * page)),
                        "any": rng.randint(0, max(1, min(most, 2 * pages * page // rows))),
                        "over": rng.choice((n, most, -3, 2 ** 31 - 1, 0))}[kind] for n in at]
        got = pool.step(None if lengths is None else i32(lengths), None if parents is None else i32(parents))
        want = plain.step(lengths, parents)
        assert got.tolist() == want, t
        same(pool, plain, mine)
        for c in mine:                                  # other tokens from now on
            c.view(-1)[:: 7] = t
        plain.caches = [c.clone() for c in mine]
        if rng.random() < 0.3:
            assert int(pool.compact()) == plain.compact()
            same(pool, plain, mine)
    assert pool.free_pages() == plain.refs().count(0)


def test_beams_share_their_prompt_and_copy_their_last_page():
    page, rows = 4, 4
    mine = caches(64, page, ("fp32",))
    pool, plain = CachePages(64, page, rows, 10, DEV, caches=mine), Plain(64, page, rows, 10, mine)
    for lengths, parents in (([10, 0, 0, 0], None), ([10, 10, 10, 10], [0, 0, 0, 0]), ([11] * 4, [0, 1, 2, 3]), ([12] * 4, [1, 1, 3, 3]),
                             ([13] * 4, [2, 2, 2, 2]), ([14] * 4, [0, 0, 1, 1]), ([6, 3, 14, 0], [0, 1, 2, 3]), ([7, 4, 15, 9], [0, 0, 2, 2])):
        assert pool.step(i32(lengths), i32(parents) if parents else None).all()
        assert all(plain.step(lengths, parents))
        same(pool, plain, mine)
    # every row's tokens are its parent's, whatever the others write behind them
    pool.fork(i32([2, 2, 2, 2]))
    plain.step(None, [2, 2, 2, 2])
    same(pool, plain, mine)
    assert pool.step(i32([15, 16, 17, 18])).all()
    # row 0 stays as it is and holds the page, so each of the others has a copy
    assert len({int(pool.table[i, 3]) for i in range(4)}) == 4
    before = mine[0][int(pool.table[0, 3]), :3].clone()
    for i in (1, 2, 3):
        mine[0][int(pool.table[i, 3]), 3] = 99.0
        assert torch.equal(mine[0][int(pool.table[i, 3]), :3], before)


def test_a_longer_holder_keeps_its_tokens():
    """Two rows of one last page, of other lengths: the shorter one never writes into the longer's."""
    mine = caches(32, 8, ("fp32",))
    for first, second in ((5, 7), (7, 5)):
        pool, plain = CachePages(32, 8, 3, 4, DEV, caches=mine), Plain(32, 8, 3, 4, mine)
        for lengths, parents in (([7, 0, 0], None), ([first, second, 0], [0, 0, -1]), ([first + 1, second + 1, 0], None)):
            got = pool.step(i32(lengths), None if parents is None else i32(parents))
            assert got.tolist() == plain.step(lengths, parents)
            same(pool, plain, mine)
        keeps = 0 if first > second else 1
        assert int(pool.table[keeps, 0]) == 0 and int(pool.table[1 - keeps, 0]) == 1


def test_a_pool_that_runs_dry():
    pool, plain = CachePages(10, 4, 5, 10, DEV), Plain(10, 4, 5, 10)
    for lengths in ([12, 20, 9, 4, 1], [12, 20, 13, 4, 8], [0, 20, 13, 4, 8], [100, 21, 13, 4, 8], [8, 8, 8, 8, 8], [9, 9, 9, 9, 9]):
        got = pool.step(i32(lengths))
        assert got.tolist() == plain.step(lengths)
        same(pool, plain)
    # sums of wants past 32 bits
    pool, plain = CachePages(5000, 1, 4096, 5000, DEV), Plain(5000, 1, 4096, 5000)
    for lengths in ([5000] * 4096, [1] * 4096, [2 ** 31 - 1] * 2000 + [1] * 2096):
        assert pool.step(i32(lengths)).tolist() == plain.step(lengths)
        same(pool, plain)


@pytest.mark.parametrize("pages", [100, 1024, 2500, 70001])
def test_compacting(pages):
    rng = random.Random(pages)
    page, rows = 2, 40
    wide = min(pages, max(8, 2 * pages // rows))
    mine = caches(pages, page, ("odd", "bf16"))
    for share in (0.0, 0.1, 0.5, 1.0):
        pool, plain = CachePages(pages, page, rows, wide, DEV, caches=mine), Plain(pages, page, rows, wide, mine)
        ids = rng.sample(range(pages), int(pages * share))
        for i, p in enumerate(ids):
            if len(plain.table[i % rows]) < wide:
                plain.table[i % rows].append(p)
        plain.lengths = [page * len(r) - (len(r) > 0 and i % page) for i, r in enumerate(plain.table)]
        table = torch.full((rows, wide), -5, dtype=torch.int64)
        for i, r in enumerate(plain.table):
            table[i, :len(r)] = torch.tensor(r, dtype=torch.int64)
        pool.load(table, torch.tensor(plain.lengths))
        same(pool, plain, mine)
        assert int(pool.compact()) == plain.compact()
        same(pool, plain, mine)
        assert int(pool.compact()) == plain.compact()                   # nothing left to move
        same(pool, plain, mine)
        lengths = [n + 3 for n in plain.lengths]
        assert pool.step(i32(lengths)).tolist() == plain.step(lengths)
        same(pool, plain, mine)
        mine = [c.clone() for c in plain.caches]


def test_layouts_of_caches():
    """Tokens behind the heads, values for a whole page, layers of one tensor, odd sizes, several groups."""
    pages, page = 30, 6
    gen = torch.Generator(device=DEV).manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    layers = rnd(5, 2, pages, page, 3, 5).half()                        # layers, key and value
    heads = rnd(pages, 4, 3, page, 9)
    scales = [rnd(pages, 7), rnd(pages)]
    flat = rnd(pages, page)
    wide = rnd(pages, 2, page, 8)[:, 1]                                 # pages with a gap
    pool = CachePages(pages, page, 4, 6, DEV, caches=[layers[i, j] for i in range(5) for j in range(2)])
    pool.add_caches([heads], token_dim=3)
    pool.add_caches(scales, token_dim=None)
    pool.add_caches([flat, wide])
    every = [layers[i, j] for i in range(5) for j in range(2)] + [flat, wide]
    by_token = every + [heads.movedim(3, 1)]
    want = [t.clone() for t in by_token]
    whole = [s.clone() for s in scales]
    assert pool.step(i32([17, 0, 0, 0])).all() and pool.step(i32([17, 17, 0, 3]), i32([0, 0, -1, 0])).all()
    assert pool.step(i32([18, 18, 0, 4])).all()
    moved = [(2, 3, 5), (0, 4, 3)]                                      # rows 0 and 1 share 0 .. 2, row 3 has 0
    assert pool.table[:, :3].tolist() == [[0, 1, 2], [0, 1, 3], [-1] * 3, [4, -1, -1]]
    for src, dst, fill in moved:
        for t in want:
            t[dst, :fill] = t[src, :fill]
        for t in whole:
            t[dst] = t[src]
    assert all(torch.equal(a, b) for a, b in zip(by_token, want)) and all(torch.equal(a, b) for a, b in zip(scales, whole))
    pool.copy_pages(i32([9, 40, 1, -1]), i32([20, 3, 21, 5]))
    for t in want + whole:
        t[20], t[21] = t[9], t[1]
    assert all(torch.equal(a, b) for a, b in zip(by_token, want)) and all(torch.equal(a, b) for a, b in zip(scales, whole))
    pool.step(i32([0, 18, 0, 4]))
    refs = pool.refs.tolist()
    used = [p for p in range(pages) if refs[p]]
    holes, movers = [p for p in range(len(used)) if not refs[p]], [p for p in used if p >= len(used)]
    pool.compact()
    for dst, src in zip(holes, movers):
        for t in want + whole:
            t[dst] = t[src]
    assert movers and all(torch.equal(a, b) for a, b in zip(by_token, want)) and all(torch.equal(a, b) for a, b in zip(scales, whole))


def test_caches_past_32_bit_offsets():
    pages, page = 40, 2
    c = torch.empty((pages, page, 1 << 26), dtype=torch.uint8, device=DEV)       # 128 MB a page
    for p in range(pages):
        c[p].fill_(p)
    pool = CachePages(pages, page, 3, pages, DEV, caches=[c])
    assert pool.step(i32([2 * pages - 3, 0, 0])).all() and pool.step(i32([2 * pages - 3, 2 * pages - 3, 0]), i32([0, 0, -1])).all()
    assert pool.step(i32([2 * pages - 2, 2 * pages - 2, 0])).all()
    assert pool.table[1, pages - 2] == pages - 1
    assert int(c[pages - 1, 0].min()) == int(c[pages - 1, 0].max()) == pages - 2
    assert int(c[pages - 1, 1].min()) == int(c[pages - 1, 1].max()) == pages - 1        # past the tokens: left as it was


def test_lengths_may_be_the_pools_own():
    pool, plain = CachePages(50, 4, 5, 8, DEV), Plain(50, 4, 5, 8)
    for lengths, parents in (([5, 9, 1, 0, 7], None), ([1, 2, 3, 4, 5], None)):
        assert pool.step(i32(lengths)).tolist() == plain.step(lengths)
    for parents in (None, [1, 0, 3, 3, 2]):
        assert pool.step(pool.lengths, None if parents is None else i32(parents)).tolist() == plain.step(list(plain.lengths), parents)
        same(pool, plain)
    assert pool.step(pool.lengths + 6).tolist() == plain.step([n + 6 for n in plain.lengths])
    same(pool, plain)


def test_state_put_back():
    pool = CachePages(200, 4, 8, 12, DEV)
    pool.step(i32([9, 7, 30, 1, 0, 4, 8, 12]))
    kept = pool.state.clone()
    first = pool.step(pool.lengths + 5, i32([2, 2, 2, 0, 1, 5, 5, 7]))
    then = pool.state.clone()
    pool.state.copy_(kept)
    again = pool.step(pool.lengths + 5, i32([2, 2, 2, 0, 1, 5, 5, 7]))
    assert torch.equal(first, again) and torch.equal(pool.state, then)


def test_captured_steps_replay():
    mine = caches(300, 4, ("bf16",))
    pool, plain = CachePages(300, 4, 12, 20, DEV, caches=mine), Plain(300, 4, 12, 20, mine)
    assert pool.step(i32([5] * 12)).all() and all(plain.step([5] * 12))
    lengths, parents = i32([5] * 12), i32(list(range(12)))
    kept = pool.state.clone()
    pool.step(lengths + 1, parents)
    pool.compact()
    pool.state.copy_(kept)
    mine[0].copy_(plain.caches[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        granted = pool.step(lengths, parents)
        live = pool.compact()
    rng = random.Random(4)
    for t in range(6):
        p = [rng.randrange(12) for _ in range(12)]
        n = [plain.lengths[q] + rng.randint(-2, 5) for q in p]
        parents.copy_(i32(p))
        lengths.copy_(i32(n))
        graph.replay()
        torch.cuda.synchronize()
        assert granted.tolist() == plain.step(n, p) and int(live) == plain.compact()
        same(pool, plain, mine)
        assert torch.equal(mine[0].float() * 2.0, plain.caches[0].float() + mine[0].float())


def test_on_a_side_stream_and_dropped_there():
    mine = caches(4000, 4, ("bf16",))
    plain = Plain(4000, 4, 200, 20, mine)
    pool = CachePages(4000, 4, 200, 20, DEV, caches=mine)
    rng = random.Random(5)
    todo = [([rng.randint(1, 40) for _ in range(200)], [rng.randrange(200) for _ in range(200)]) for _ in range(4)]
    todo = [(i32(n), i32(p), n, p) for n, p in todo]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(10_000_000)
        got = [pool.step(n, p) for n, p, _, _ in todo]
        table = pool.table.clone()
        sizes = pool.state.numel() * 4, pool._scratch.numel()
        del pool
    junk = [torch.full((n,), 0xFF, dtype=torch.uint8, device=DEV) for n in sizes for _ in range(4)]
    side.synchronize()
    for g, (_, _, n, p) in zip(got, todo):
        assert g.tolist() == plain.step(n, p)
    assert [[v for v in row if v >= 0] for row in table.tolist()] == plain.table
    assert torch.equal(mine[0], plain.caches[0]) and all(int(j.min()) == 0xFF for j in junk)


def test_refusals():
    pool = CachePages(20, 4, 3, 6, DEV)
    for call in (lambda: pool.step(torch.zeros(3, device=DEV)), lambda: pool.step(i32([1, 2])), lambda: pool.step(i32([1, 2, 3]).cpu()),
                 lambda: pool.step(None, i32([0, 1])), lambda: pool.copy_pages(i32([1]), i32([1, 2])),
                 lambda: pool.copy_pages(i32([[1]]), i32([1])),
                 lambda: pool.load(torch.zeros(3, 5), torch.zeros(3)), lambda: pool.load(torch.zeros(3, 6), torch.tensor([25, 0, 0])),
                 lambda: pool.load(torch.zeros(3, 6), torch.tensor([-1, 0, 0])), lambda: pool.load(torch.full((3, 6), 20), torch.tensor([1, 0, 0])),
                 lambda: pool.load(torch.full((3, 6), 3), torch.tensor([5, 0, 0])),
                 lambda: pool.add_caches([torch.zeros(19, 4, 2, device=DEV)]), lambda: pool.add_caches([torch.zeros(20, 5, 2, device=DEV)]),
                 lambda: pool.add_caches([torch.zeros(20, 4, 2)]), lambda: pool.add_caches([torch.zeros(20, 4, 2, device=DEV).transpose(1, 2)], 2),
                 lambda: pool.add_caches([torch.zeros(20, 2, 3, 4, 2, device=DEV).transpose(1, 2)], 3),
                 lambda: pool.add_caches([torch.zeros(4, 2, device=DEV).expand(20, 4, 2)]), lambda: pool.add_caches([torch.zeros(20, device=DEV)]),
                 lambda: pool.add_caches([torch.zeros(20, 4, i + 1, device=DEV) for i in range(9)])):
        with pytest.raises(ValueError):
            call()
    pool.copy_pages(i32([]), i32([]))
    assert pool.step(i32([24, 0, 25])).tolist() == [True, True, False]
