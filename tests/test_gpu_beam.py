"""Beam search's selection on an MI355X against 64 bits.

A score is score + (x - top) - log(sum), one rounding at the end: half a unit, 2^-24 of it.  Before
that only the sum of exp(x - top) is not in 64 bits: each weight's argument is rounded three times
(the difference, the product with log2 e and that constant), 3 * 2^-24 of |x - top| each at most,
its exponential by a unit (2^-23), 32 of them are added in fp32 (4 sums of 8, then 2 more: 10 *
2^-24), and the threads' sums are scaled once more to the row's maximum (as the arguments).  In all
the logarithm is off by at most 2^-24 * (6 * mean |x - top| + 16), the mean over the weights.

Continuations whose exact totals differ by less than the two bounds may change places.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from fie_amd.beam import Beams, beam_step, first_beams

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
UNIT = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
LOW, LARGEST = -np.inf, float(np.finfo(np.float32).max)


def oracle(logits, beams, eos=(), length_penalty=1.0, early_stopping=False, min_tokens=0, max_tokens=0, pad=0):
    """The step in 64 bits: per request the continuations in order, and what comes of them."""
    x = logits.double().cpu().numpy()
    scores, lengths, done, pool, ends = (t.cpu().numpy() for t in beams)
    R, K = scores.shape
    x = np.minimum(np.where(np.isnan(x), LOW, x), LARGEST).reshape(R, K, -1)
    V = x.shape[2]
    out = dict(scores=np.full((R, K), LOW), tokens=np.full((R, K), pad), parents=np.arange(R * K).reshape(R, K).copy(),
               lengths=lengths + ~done, done=done.copy(), pool=pool.astype(np.float64), ends=ends.copy(), off=np.zeros((R, K)),
               all=[None] * R, total=[None] * R)
    for r in range(R):
        if done[r]:
            continue
        total, off = np.full((K, V), LOW), np.zeros(K)
        for b in range(K):
            top = x[r, b].max()
            if not scores[r, b] > LOW or top == LOW:
                continue
            d = x[r, b] - top
            w = np.exp(d)
            total[b] = float(scores[r, b]) + (d - np.log(w.sum()))
            off[b] = UNIT * (6 * (w * np.where(w > 0, -d, 0.0)).sum() / w.sum() + 16)
        flat = total.reshape(-1)
        keep = min(flat.size, 4 * K + K * len(eos) + 8)
        # by total, then beam, then the larger logit, then the lower token
        some = np.nonzero(flat >= np.partition(flat, flat.size - keep)[flat.size - keep])[0]
        some = some[flat[some] > LOW]
        order = some[np.lexsort((some % V, -x[r].reshape(-1)[some], some // V, -flat[some]))]
        length = int(lengths[r]) + 1
        ending = np.isin(order % V, eos)
        order = order[~ending] if length < min_tokens else order
        ending = np.isin(order % V, eos) | bool(max_tokens and length >= max_tokens)
        scale = float(length) ** length_penalty
        new = [(flat[c] / scale, (length, r * K + c // V, c % V)) for c in order[:K][ending[:K]]]
        live = order[~ending][:K]
        entries = [(float(v), tuple(e)) for v, e in zip(pool[r], ends[r])] + [(float(np.float32(v)), e) for v, e in new]
        entries = sorted(entries, key=lambda e: -e[0])[:K]
        out["pool"][r], out["ends"][r] = [v for v, _ in entries], [e for _, e in entries]
        full = entries[-1][0] > LOW
        best = np.float32(flat[live[0]] / scale) if len(live) else LOW
        out["done"][r] = not len(live) or (full and (early_stopping or entries[-1][0] >= best))
        out["all"][r], out["total"][r] = order, total
        out["off"][r] = off
        if not out["done"][r]:
            n = len(live)
            out["scores"][r, :n], out["tokens"][r, :n] = flat[live], live % V
            out["parents"][r, :n] = r * K + live // V
    return out


def check(logits, beams, got=None, **kw):
    got = beam_step(logits, beams, **kw) if got is None else got
    kw.pop("inplace", None)
    kw.pop("history", None)
    want = oracle(logits, beams, **kw)
    R, K = beams.scores.shape
    b = got.beams
    assert got.tokens.dtype == torch.int64 and got.parents.dtype == torch.int32
    tokens, parents = got.tokens.cpu().numpy().reshape(R, K), got.parents.cpu().numpy().reshape(R, K)
    scores, pool, ends = b.scores.cpu().numpy(), b.pool.cpu().numpy(), b.ends.cpu().numpy()
    np.testing.assert_array_equal(b.lengths.cpu().numpy(), want["lengths"])
    np.testing.assert_array_equal(b.done.cpu().numpy(), want["done"])
    for r in range(R):
        off = 2 * want["off"][r].max()
        for j in range(K):
            if (tokens[r, j], parents[r, j]) != (want["tokens"][r, j], want["parents"][r, j]):
                # two that differ by less than the bounds
                mine = want["total"][r][parents[r, j] - r * K, tokens[r, j]]
                assert abs(mine - want["scores"][r, j]) <= off, (r, j, mine, want["scores"][r, j])
        ok = np.isfinite(want["scores"][r])
        np.testing.assert_array_equal(np.isfinite(scores[r]), ok)
        assert (np.abs(scores[r] - want["scores"][r])[ok] <= (UNIT * np.abs(want["scores"][r]) * 1.01 + off)[ok]).all()
        ok = np.isfinite(want["pool"][r])
        np.testing.assert_array_equal(np.isfinite(pool[r]), ok)
        assert (np.abs(pool[r] - want["pool"][r])[ok] <= (2 * UNIT * np.abs(want["pool"][r]) + off)[ok]).all()
        if off == 0 or not (np.abs(np.diff(want["pool"][r][ok])) <= off).any():
            np.testing.assert_array_equal(ends[r], want["ends"][r])
    return got


def rows(seed, n, V, dtype=torch.float32, spread=3.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (spread * torch.randn(n, V, generator=gen, device=DEV)).to(dtype)


def some_beams(seed, R, K, filled=True):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    b = first_beams(R, K, DEV)
    b.scores.copy_((-5.0 * torch.rand(R, K, generator=gen, device=DEV)).sort(1, descending=True).values)
    b.lengths.copy_(torch.randint(1, 50, (R,), generator=gen, device=DEV))
    if filled:
        n = torch.randint(0, K + 1, (R, 1), generator=gen, device=DEV)
        v = (-2.0 * torch.rand(R, K, generator=gen, device=DEV) - 0.2).sort(1, descending=True).values
        has = torch.arange(K, device=DEV) < n
        b.pool.copy_(torch.where(has, v, b.pool))
        b.ends.copy_(torch.where(has[:, :, None], torch.randint(0, 99, (R, K, 3), generator=gen, device=DEV).int(), b.ends))
    return b


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R, K, V", [(1, 1, 1), (1, 1, 2), (1, 4, 3), (2, 3, 7), (1, 2, 63), (3, 5, 100), (2, 8, 255), (1, 4, 2047),
                                     (2, 2, 8191), (1, 3, 8192), (1, 4, 8193), (5, 4, 20001), (3, 16, 50001), (1, 64, 5000),
                                     (2, 33, 32768), (1, 4, 151936), (70, 8, 9000), (300, 7, 301), (1, 5, 524288)])
def test_sizes(R, K, V, dtype):
    print(f"  case: {R} x {K} x {V} {dtype}", flush=True)
    eos = sorted({V // 2, V - 1})[:1 if V < 3 else 2]
    check(rows(R + K + V, R * K, V, dtype), some_beams(V, R, K), eos=eos)
    check(rows(R * K + V, R * K, V, dtype, 0.01), some_beams(V + 1, R, K), eos=(), length_penalty=0.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_first_step_reads_a_row_a_request(dtype):
    """Rows of beams that are not there may hold anything."""
    R, K, V = 4, 6, 3001
    x = rows(1, R * K, V, dtype)
    x.view(R, K, V)[:, 1:] = float("nan")
    b = first_beams(R, K, DEV)
    got = check(x, b, eos=[5])
    assert (got.parents.view(R, K) == torch.arange(R, device=DEV)[:, None] * K).all()
    assert torch.isfinite(got.beams.scores).all()
    # and as many steps as it takes
    for i in range(4):
        got = check(rows(10 + i, R * K, V, dtype), got.beams, eos=[5, 77], early_stopping=bool(i % 2))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [100, 2500, 20001, 70000])
def test_equal_logits_go_by_beam_and_index(V, dtype):
    """All continuations of a beam alike: the lowest tokens, of the better beam first."""
    K = 6
    x = torch.full((2 * K, V), 1.5, device=DEV).to(dtype)
    b = some_beams(3, 2, K, filled=False)
    got = check(x, b)
    assert got.tokens.view(2, K).tolist() == [list(range(K))] * 2
    assert got.parents.view(2, K).tolist() == [[0] * K, [K] * K]
    # equal beams: the lower one, as long as it has any
    b.scores.fill_(-1.0)
    got = check(x, b, eos=[1, 2])
    assert got.tokens.view(2, K).tolist() == [[0, 3, 4, 5, 6, 7]] * 2 and (got.parents.view(2, K)[1] == K).all()


@pytest.mark.parametrize("V", [9000, 40000, 151936])
def test_logits_in_rising_and_falling_order(V):
    """Every tile better than the one before it, and ties across tiles."""
    up = torch.arange(V, device=DEV).float()
    x = torch.stack([up * 1e-4, -up * 1e-4, (up // 5000), -(up // 3000), (up % 7), torch.where(up == V - 1, 9.0, 1.0)])
    check(x, some_beams(5, 1, 6), eos=[V - 1, 0])
    check(x.repeat(4, 1), some_beams(6, 3, 8), eos=[V - 2])


@pytest.mark.parametrize("dtype", DTYPES)
def test_masks(dtype):
    """-inf does not exist, the type's lowest value does; rows with nothing left; NaN and infinities."""
    V, K, low = 9001, 4, torch.finfo(dtype).min
    x = rows(7, 8 * K, V, dtype).view(8, K, V)
    x[0] = float("-inf")                                # nothing: done
    x[1, :, 3:] = float("-inf")                         # three tokens a beam
    x[2, 1:] = float("-inf")                            # one beam of four
    x[2, 0, 2:] = float("-inf")                         # and of it two tokens
    x[3] = low                                          # all alike
    x[4, :, 10:] = low
    x[4, :, 0] = float("-inf")
    x[5, :, ::3] = float("nan")
    x[6, 0, 100] = x[6, 0, 8200] = x[6, 2, 17] = float("inf")
    x[7, 1] = float("nan")
    x[7, 0, 1:] = float("-inf")
    got = check(x.view(-1, V), some_beams(8, 8, K), eos=[1])
    assert got.beams.done[0] and (got.parents[:K].tolist() == list(range(K)))
    assert torch.isfinite(got.beams.scores[2]).sum() <= 2


def test_no_such_beams_and_requests_that_are_through():
    R, K, V = 6, 5, 2222
    b = some_beams(9, R, K)
    b.scores[1, 2:] = float("-inf")
    b.scores[2] = float("-inf")
    b.scores[3, 0] = float("nan")
    b.done[4] = True
    x = rows(9, R * K, V)
    x.view(R, K, V)[4] = float("nan")
    got = check(x, b, eos=[3])
    assert torch.equal(got.beams.pool[4], b.pool[4]) and torch.equal(got.beams.ends[4], b.ends[4])
    assert got.beams.lengths[4] == b.lengths[4] and got.beams.done[2]
    assert (got.tokens.view(R, K)[4] == 0).all()
    assert (beam_step(x, b, pad=77).tokens.view(R, K)[4] == 77).all()


@pytest.mark.parametrize("alpha", [0.0, 0.7, 1.0, 2.5, -1.0])
@pytest.mark.parametrize("early", [False, True])
def test_ending(alpha, early):
    """Endings among the best, not among them, many at once, at a pool with room and without."""
    R, K, V = 40, 4, 500
    x = rows(11, R * K, V)
    eos = [7, 400, 401]
    near = x.amax(1, keepdim=True) - 2.0 * torch.rand(R * K, 3, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    x[:, eos] = near
    b = some_beams(12, R, K)
    got = check(x, b, eos=eos, length_penalty=alpha, early_stopping=early)
    assert got.beams.done.any() or not early
    assert (got.beams.ends != b.ends).any()
    check(x, b, eos=eos, length_penalty=alpha, early_stopping=early, min_tokens=25)
    got = check(x, b, eos=eos, length_penalty=alpha, early_stopping=early, max_tokens=20)
    assert got.beams.done[b.lengths >= 19].all()


@pytest.mark.parametrize("R, K, V, E", [(1, 64, 151936, 0), (1, 64, 151936, 16), (2, 40, 100001, 3), (1, 33, 524288, 16)])
def test_more_candidates_than_are_ranked_at_once(R, K, V, E):
    """Lists of many spans and beams, taken one by one; and lists of equal totals, which no bound cuts."""
    print(f"  case: {R} x {K} x {V}, {E} eos", flush=True)
    eos = [V // 3 + i for i in range(E)]
    x = rows(V + K, R * K, V, torch.bfloat16)
    if E:
        x[:, eos] = x.amax(1, keepdim=True) - torch.rand(R * K, E, device=DEV).bfloat16()
    b = some_beams(V, R, K)
    check(x, b, eos=eos)
    b.scores.fill_(-2.0)
    check(x[:1].expand(R * K, V), b, eos=eos, max_tokens=60)
    check(torch.zeros(R * K, V, device=DEV), b, eos=eos)


def test_equal_beams_past_the_ranked_list():
    """As many equal totals as a request has candidates: by beam, then token."""
    for K, V in ((16, 60000), (30, 20001)):
        b = some_beams(2, 3, K)
        b.scores.fill_(-1.0)
        x = rows(5, 1, V, torch.float16).expand(3 * K, V)
        got = check(x, b, eos=[4])
        if V % 8 == 0:
            # (rows that begin at other addresses are summed in another order: their logarithms are
            # equal within the bound above, and check() has looked at that)
            assert (got.parents.view(3, K)[:, :2] - torch.tensor([[0], [K], [2 * K]], device=DEV) == torch.tensor([0, 1], device=DEV)).all()
        check(torch.ones(3 * K, V, device=DEV), b, eos=[0, 2])


def test_many_eos_and_a_vocabulary_of_nothing_else():
    got = check(rows(13, 8, 16), some_beams(13, 2, 4), eos=range(16))
    assert got.beams.done.all()
    check(rows(14, 64, 4000), some_beams(14, 1, 64), eos=range(100, 116))
    check(rows(15, 6, 20), some_beams(15, 1, 6), eos=range(16))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("at, pad", [(0, 1), (1, 3), (3, 5), (8, 8), (13, 0)])
def test_strides_and_alignment(at, pad, dtype):
    R, K, V = 2, 3, 9999
    wide = torch.full((R * K, at + V + pad), 1e4, device=DEV).to(dtype)
    wide[:, at:at + V] = rows(16, R * K, V, dtype)
    check(wide[:, at:at + V], some_beams(16, R, K), eos=[V - 1])
    check(wide[:, at:at + V].t().contiguous().t(), some_beams(16, R, K), eos=[0])


def test_past_32_bit_offsets():
    """Rows more than 2^32 bytes apart."""
    R, K, V, step = 2, 2, 5000, 3 * (1 << 30) // 2 + 1
    room = torch.empty(3 * step + V, dtype=torch.bfloat16, device=DEV)
    x = room.as_strided((R * K, V), (step, 1))
    x.copy_(rows(21, R * K, V, torch.bfloat16))
    check(x, some_beams(21, R, K), eos=[7])


def test_inplace_and_history():
    R, K, V, T = 3, 4, 700, 5
    rows_ = R * K
    old = some_beams(17, R, K)
    old.lengths.copy_(torch.tensor([0, 2, 4]))
    old.done[1] = True
    x = rows(17, rows_, V)
    want = beam_step(x, old, eos=[9])
    mine = Beams(*(t.clone() for t in old))
    history = tuple(torch.full((T, rows_), -7, dtype=torch.int32, device=DEV) for _ in range(2))
    got = beam_step(x, mine, eos=[9], inplace=True, history=history)
    assert got.beams.scores is mine.scores
    for a, b in zip(got.beams, want.beams):
        assert torch.equal(a, b)
    assert torch.equal(got.tokens, want.tokens) and torch.equal(got.parents, want.parents)
    for h, v in zip(history, (got.tokens.int(), got.parents)):
        seen = h.view(T, R, K)
        for r, t in ((0, 0), (2, 4)):
            assert torch.equal(seen[t, r], v.view(R, K)[r])
            seen[t, r] = -7
        assert (h == -7).all()


def test_repeats_are_the_same_bits():
    x = rows(18, 40, 30001, torch.bfloat16)
    b = some_beams(18, 5, 8)
    first = beam_step(x, b, eos=[4])
    for _ in range(5):
        again = beam_step(x, b, eos=[4])
        assert all(torch.equal(s, t) for s, t in zip((*first.beams, *first[1:]), (*again.beams, *again[1:])))


def test_a_captured_step_replays():
    R, K, V = 4, 4, 20001
    x = rows(19, R * K, V, torch.float16)
    start = some_beams(19, R, K)
    b = Beams(*(t.clone() for t in start))
    beam_step(x, b, eos=[3])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = beam_step(x, b, eos=[3], inplace=True)
    for i in range(4):
        x.copy_(rows(30 + i, R * K, V, torch.float16))
        for t, s in zip(b, start):
            t.copy_(s)
        want = beam_step(x, start, eos=[3])
        graph.replay()
        torch.cuda.synchronize()
        for s, t in zip((*want.beams, *want[1:]), (*got.beams, *got[1:])):
            assert torch.equal(s, t)


def test_on_a_side_stream():
    x, b = rows(20, 32, 50001), some_beams(20, 8, 4)
    want = beam_step(x, b, eos=[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(5_000_000)
        got = beam_step(x, b, eos=[1])
        again = beam_step(x, got.beams, eos=[1])
    other = beam_step(x, want.beams, eos=[1])
    side.synchronize()
    assert torch.equal(got.tokens, want.tokens) and torch.equal(again.beams.scores, other.beams.scores)
