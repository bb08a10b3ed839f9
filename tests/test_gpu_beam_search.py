"""States gathered by their parents, and a whole search, on an MI355X."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from fie_amd.beam import MAX_STATES, BeamSearch, reorder_states

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.uint8, torch.float64, torch.bool])
@pytest.mark.parametrize("width", [1, 2, 3, 7, 8, 15, 16, 17, 31, 64, 1000, 4096, 8191, 16385, 40000])
def test_widths(width, dtype):
    gen = torch.Generator(device=DEV).manual_seed(width)
    for rows in (1, 2, 13):
        states = [torch.randint(0, 2 if dtype == torch.bool else 200, (rows, width), generator=gen, device=DEV).to(dtype)
                  for _ in range(3)]
        parents = torch.randint(0, rows, (rows,), generator=gen, device=DEV, dtype=torch.int32)
        room = [torch.zeros(rows + 2, width, dtype=dtype, device=DEV) for _ in states]
        got = reorder_states(states, parents)
        again = reorder_states(states, parents, out=[r[1:-1] for r in room])
        for s, g, a, r in zip(states, got, again, room):
            assert torch.equal(g, s[parents.long()]) and torch.equal(a, g)
            assert (r[0] == 0).all() and (r[-1] == 0).all()             # rows around, left as they were


@pytest.mark.parametrize("shift", [0, 1, 2, 3, 5, 8, 13])
def test_alignment_and_strides(shift):
    """Rows at any address, sources and outputs shifted against each other."""
    rows, width = 9, 5000
    gen = torch.Generator(device=DEV).manual_seed(shift)
    parents = torch.randint(0, rows, (rows,), generator=gen, device=DEV, dtype=torch.int32)
    for pad in (0, 1, 6, 16):
        src = torch.randint(0, 255, (rows, shift + width + pad), generator=gen, device=DEV, dtype=torch.uint8)
        dst = torch.full((rows, width + 40), 7, dtype=torch.uint8, device=DEV)
        for at in (0, 1, 4, 15, 16):
            dst.fill_(7)
            reorder_states([src[:, shift:shift + width]], parents, out=[dst[:, at:at + width]])
            assert torch.equal(dst[:, at:at + width], src[parents.long(), shift:shift + width])
            assert (dst[:, :at] == 7).all() and (dst[:, at + width:] == 7).all()


def test_shapes_many_tensors_and_odd_parents():
    gen = torch.Generator(device=DEV).manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    states = [rnd(6, 3, 5), rnd(6), rnd(6, 2, 0), rnd(8, 4, 4).bfloat16(), rnd(4, 6).t(), rnd(1, 5).expand(6, 5)]
    states += [rnd(6, 11 + i) for i in range(2 * MAX_STATES)]
    parents = torch.tensor([5, 5, 0, -1, 100, 2], dtype=torch.int32, device=DEV)
    at = [5, 5, 0, 3, 4, 2]                             # a parent that is no row: the row's own
    parents[4] = 2 ** 31 - 1
    for s, g in zip(states, reorder_states(states, parents)):
        assert g.is_contiguous() and torch.equal(g, s[at])
    assert reorder_states([], parents) == []
    assert reorder_states([rnd(6, 4)], parents[:0])[0].shape == (0, 4)
    assert torch.equal(reorder_states([states[0]], parents[:2])[0], states[0][[5, 5]])
    strided = torch.stack([parents, parents + 1], 1)[:, 0]
    assert torch.equal(reorder_states([states[0]], strided)[0], states[0][at])


def test_states_past_32_bit_offsets():
    rows, width = 5, 1 << 30
    s = torch.empty((rows, width), dtype=torch.uint8, device=DEV)
    for i in range(rows):
        s[i] = 10 + i
    got = reorder_states([s], torch.tensor([4, 0, 4, 3, 1], dtype=torch.int32, device=DEV))[0]
    assert [(int(r.min()), int(r.max())) for r in got] == [(14, 14), (10, 10), (14, 14), (13, 13), (11, 11)]


def test_refusals():
    s, p = torch.zeros(4, 8, device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV)
    for states, parents, out in (([s], p.long(), None), ([s], p[None], None), ([s], p.cpu(), None), ([s.cpu()], p, None),
                                 ([s[:3]], p, None), ([s], p, []), ([s], p, [s]), ([s], p, [s.half()]), ([s], p, [s[:2]]),
                                 ([s], p, [torch.zeros(8, 4, device=DEV).t()]), ([s], p, [torch.zeros(8, device=DEV).expand(4, 8)]),
                                 ([s[0, 0]], p, None)):
        with pytest.raises(ValueError):
            reorder_states(states, parents, out)
    big = torch.zeros(6, 8, device=DEV)
    with pytest.raises(ValueError):
        reorder_states([big[:4]], p, [big[2:]])
    assert reorder_states([big[:2]], p[:2], [big[2:4]])[0].shape == (2, 8)


def tables(seed, V, steps):
    """Log-probabilities of a token after another, for each of some steps: a model to search in."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return torch.log_softmax(2.0 * torch.randn(steps, V, V, generator=gen, device=DEV), 2)


def searched(t, start, beams, eos, alpha, steps):
    """The same search, on the host in 64 bits."""
    t = t.double().cpu().numpy()
    live, pool = [(0.0, [start])], []
    for n in range(1, steps + 1):
        every = sorted(((s + t[n - 1, w[-1], v], w + [v]) for s, w in live for v in range(t.shape[2])), key=lambda e: -e[0])
        pool += [(s / n ** alpha, w) for s, w in every[:beams] if w[-1] == eos or n == steps]
        pool = sorted(pool, key=lambda e: -e[0])[:beams]
        live = [e for e in every if e[1][-1] != eos][:beams]
        if n == steps or (len(pool) == beams and pool[-1][0] >= live[0][0] / n ** alpha):
            return [(v, w[1:]) for v, w in pool]


@pytest.mark.parametrize("beams, alpha", [(1, 1.0), (3, 0.0), (4, 1.0), (7, 2.0)])
def test_a_whole_search(beams, alpha):
    V, steps, R, eos = 40, 12, 5, 3
    t = tables(beams, V, steps)
    search = BeamSearch(DEV, R, beams, max_tokens=steps, eos=[eos], length_penalty=alpha)
    token = torch.arange(5, 5 + R, device=DEV).repeat_interleave(beams)
    memory = token.clone()[:, None].repeat(1, 3)                        # a state that goes with the beams
    for n in range(steps):
        if search.all_done():
            break
        got = search.step(t[n, token])
        token = got.tokens
        memory = reorder_states([memory], got.parents)[0]
        memory[:, 1] = token
    assert search.all_done()
    for r in range(R):
        answers = search.answers(r)
        want = searched(t, 5 + r, beams, eos, alpha, steps)
        assert [a.tokens for a in answers] == [w for _, w in want] and all(a.ended for a in answers)
        # fp32 scores of `steps` additions, each rounded by half a unit of at most |score|, and a quotient
        np.testing.assert_allclose([a.value for a in answers], [v for v, _ in want], rtol=(steps + 2) * 2.0 ** -24)
    assert (memory[:, 0] == torch.arange(5, 5 + R, device=DEV).repeat_interleave(beams)).all()


def test_slots_that_fill_up_the_batch():
    """Stopped slots are not read, change nothing, and begin when they are asked to."""
    V, beams = 50, 3
    x = torch.randn(3 * beams, V, device=DEV, generator=torch.Generator(device=DEV).manual_seed(3))
    alone, search = BeamSearch(DEV, 1, beams, max_tokens=5, eos=[1]), BeamSearch(DEV, 3, beams, max_tokens=5, eos=[1])
    search.stop([0, 2])
    x[:beams] = x[2 * beams:] = float("nan")
    for _ in range(3):
        got, want = search.step(x), alone.step(x[beams:2 * beams].clone())
        assert got.parents[:beams].tolist() == list(range(beams)) and (got.tokens[2 * beams:] == 0).all()
        assert torch.equal(got.tokens[beams:2 * beams], want.tokens) and torch.equal(got.parents[beams:2 * beams] - beams, want.parents)
    assert search.answers(0) == [] and search.beams.lengths.tolist() == [0, 3, 0]
    search.restart([2])
    x[2 * beams:] = 0.0
    assert search.step(x).parents[2 * beams:].tolist() == [2 * beams] * beams
    search.stop([])
    search.stop([1])
    assert not [a for a in search.answers(1) if not a.ended]


def test_slots_begin_anew():
    V, steps, beams = 30, 6, 3
    t = tables(9, V, steps)
    search = BeamSearch(DEV, 2, beams, max_tokens=steps, eos=[1])
    alone = BeamSearch(DEV, 1, beams, max_tokens=steps, eos=[1])
    token = torch.full((6,), 4, device=DEV)
    for n in range(2):
        token = search.step(t[n, token]).tokens
    assert len(search.answers(1)) >= beams and not search.answers(1)[-1].ended
    assert len(search.answers(1)[-1].tokens) == 2
    search.restart([1])
    assert search.answers(1) == []
    mine = torch.full((3,), 8, device=DEV)
    token[3:] = 8
    for n in range(4):
        logits = torch.cat([t[n + 2, token[:3]], t[n, token[3:]]])
        token = search.step(logits).tokens
        mine = alone.step(t[n, mine]).tokens
    # Rows of 120 bytes begin at other addresses in another batch, so the order of their fp32 sums is
    # another: a step's log-sum is off by up to 2^-24 (6 mean |x - top| + 16), the mean at most log 30
    # = 3.4, its score's rounding by 2^-24 |score| with |score| < 4; four steps on either side, and the
    # values are quotients by 4 and less.
    got, want = search.answers(1), alone.answers(0)
    assert [(a.tokens, a.ended) for a in got] == [(a.tokens, a.ended) for a in want]
    np.testing.assert_allclose([a.value for a in got], [a.value for a in want], rtol=0, atol=2 * 4 * 41 * 2.0 ** -24)
    assert search.beams.done[0]                         # six tokens
    search.restart([])
    for bad in ([2], [-1]):
        for call in (search.restart, search.stop):
            with pytest.raises(ValueError):
                call(bad)
    with pytest.raises(ValueError):
        search.answers(2)
