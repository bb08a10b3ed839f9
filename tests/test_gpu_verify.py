"""Verification of drafted tokens on an MI355X against a plain 64-bit implementation.

Kept sets and the last rows' draws come from the canonical oracle; probabilities are its
kept weights in 64 bits.  Tests of drafts and draws of refusals are placed at least 2e-5
(relative for a test, of p's mass where it is over q for a draw) from where they change: p
is an fp32 product of an fp32 weight, an fp32 exponential and an fp32 quotient, each within
2^-22 or so of its 64-bit value, and q is exact.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import oracle as O
from fie_amd import _lib
from fie_amd.runtime.sampling import SamplingParams
from fie_amd.verify import MAX_DRAFTS, DraftVerifier

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
MARGIN = 2e-5

MIXED = [SamplingParams(), SamplingParams(temperature=1.0), SamplingParams(temperature=0.8, top_k=5),
         SamplingParams(temperature=0.7, top_p=0.9), SamplingParams(temperature=1.3, min_p=0.05, top_p=0.95),
         SamplingParams(temperature=0.9, top_k=40, top_p=0.8)]


@pytest.fixture(scope="module")
def verifier():
    return DraftVerifier(DEV)


def plain(x, params, lens, ids, probs, rng, contexts=None):
    """(uniforms, tokens, accepted, p of the drafts) of fp32 logits x, in 64 bits, with the
    uniforms moved off the places where an answer changes."""
    V = x.shape[1]
    rows = [p for p, n in zip(params, lens) for _ in range(n + 1)]
    u = rng.random(len(rows))
    res = O.resolve(rows, V)
    ctx = None
    if contexts is not None:
        at, ctx = 0, []
        for c, n in zip(contexts, lens):
            ctx += [list(c) + ids[at:at + j].tolist() for j in range(n + 1)]
            at += n
    draw = u.copy()
    ref = O.canonical_step(x, res, draw, contexts=ctx, want_kept=True)
    zero = O.canonical_step(x, res, draw * 0, contexts=ctx)      # most likely tokens
    top = max(lens, default=0)
    tokens = np.full((len(lens), top + 1), -1, np.int64)
    accepted = np.zeros(len(lens), np.int32)
    pds = np.zeros(int(sum(lens)))
    first = row = 0
    for r, n in enumerate(lens):
        took, out = 0, None
        for j in range(n + 1):
            y = (ref.penalized[row + j] / res.scale[row + j]).astype(np.float64)
            if res.greedy[row + j]:
                p = np.zeros(V)
                p[zero.tokens[row + j]] = 1.0
            else:
                with np.errstate(invalid="ignore"):
                    p = np.exp(y - y[np.isfinite(y)].max()) if np.isfinite(y).any() else np.zeros(V)
                p = np.where(ref.kept[row + j] > 0, np.nan_to_num(p, nan=0.0), 0.0)
                p = p / p.sum() if p.sum() else p
            if j == n:
                if out is None:
                    out = int(ref.tokens[row + j])
                break
            d = int(ids[first + j])
            ok = 0 <= d < V
            pd = p[d] if ok else 0.0
            pds[first + j] = pd
            q = np.zeros(V)
            if probs is None:
                if ok:
                    q[d] = 1.0
            else:
                q = np.nan_to_num(probs[first + j].astype(np.float64), nan=0.0, posinf=np.inf)
                q = np.maximum(q, 0.0)
            qd = q[d] if ok else 0.0
            if abs(u[row + j] * qd - pd) <= MARGIN * max(pd, qd):
                u[row + j] = 0.0 if pd > 0 else 0.5
            if out is not None:
                continue
            if u[row + j] * qd < pd:
                took += 1
                continue
            rest = np.cumsum(np.maximum(p - q, 0.0))
            if rest[-1] < 1e-9 or res.greedy[row + j] or not ok and not p.sum():
                out = int(zero.tokens[row + j])
                if res.greedy[row + j]:
                    assert out == zero.tokens[row + j]
                continue
            t = int(np.searchsorted(rest, u[row + n] * rest[-1], side="right"))
            lo, hi = (rest[t - 1] if t else 0.0) / rest[-1], rest[t] / rest[-1]
            near = MARGIN * p[p > q].sum() / rest[-1]
            if min(u[row + n] - lo, hi - u[row + n]) < near:
                wide = np.diff(rest, prepend=0.0) / rest[-1] >= 4 * near
                assert wide.any()
                t = int(rng.choice(np.nonzero(wide)[0]))
                u[row + n] = ((rest[t - 1] if t else 0.0) + rest[t]) / (2 * rest[-1])
            out = t
        tokens[r, :took] = ids[first:first + took]
        tokens[r, took] = out
        accepted[r] = took
        first += n
        row += n + 1
    return u, tokens, accepted, pds


def make(seed, requests, lens, V, dtype, drafted, kind="peaked"):
    """Logits [rows, V], draft ids and probabilities (fp32, a noisy copy of the target's)."""
    gen = torch.Generator().manual_seed(seed)
    rows, drafts = sum(lens) + requests, sum(lens)
    x = 3.0 * torch.randn(rows, V, generator=gen)
    if kind == "masked":                 # -inf and the type's lowest value in most places
        x[torch.rand(rows, V, generator=gen) < 0.7] = float("-inf")
        x[torch.rand(rows, V, generator=gen) < 0.2] = torch.finfo(dtype).min
        x[:, V // 2] = 1.0
    x = x.to(dtype)
    last = np.zeros(rows, bool)
    last[np.cumsum(np.array(lens) + 1) - 1] = True
    y = x.float()[torch.from_numpy(~last)]
    q = torch.softmax(torch.nan_to_num(y + torch.randn(drafts, V, generator=gen), neginf=-1e30), 1)
    ids = torch.multinomial(q, 1, generator=gen)[:, 0] if drafts else torch.zeros(0, dtype=torch.int64)
    return x, ids, (q if drafted else None)


def check(verifier, x, params, lens, ids, probs, seed, contexts=None, transform=None):
    V = x.shape[1]
    print(f"  case: lens={lens[:8]} vocab={V} dtype={x.dtype} probs={None if probs is None else probs.dtype}", flush=True)
    pq = None if probs is None else probs.float().numpy()
    u, tokens, accepted, pds = plain(x.float().numpy(), params, lens, ids.numpy(), pq, np.random.default_rng(seed), contexts)
    drafts, at = [], 0
    for n in lens:
        drafts.append(ids[at:at + n].tolist())
        at += n
    plan = verifier.plan(params, lens, V, contexts, drafts)
    g = [x.to(DEV), ids.to(DEV), torch.from_numpy(u).to(DEV), None if probs is None else probs.to(DEV)]
    if transform is not None:
        g = transform(g)
    got = verifier.verify(plan, *g)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(got.accepted.cpu().numpy(), accepted)
    np.testing.assert_array_equal(got.tokens.cpu().numpy(), tokens)
    # fp32 products: relative 2^-20; weights are floored at 2^-40 of their tile's largest
    np.testing.assert_allclose(got.draft_probs.cpu().numpy(), pds, rtol=2e-6, atol=2.0 ** -38)
    return got, accepted, tokens


LENS = [3, 0, 5, 1, 2, 4, 0, 2, 1, 3, 2, 1]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("draft", [None, torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 37, 2049, 20001])
def test_against_64_bits(verifier, dtype, draft, V):
    x, ids, q = make(V, 12, LENS, V, dtype, draft is not None)
    check(verifier, x, (MIXED * 2)[:12], LENS, ids, None if q is None else q.to(draft), V + 1)


@pytest.mark.parametrize("draft", [None, torch.float32])
def test_masked_logits(verifier, draft):
    for V in (50, 9000):
        x, ids, q = make(7, 12, LENS, V, torch.bfloat16, draft is not None, kind="masked")
        check(verifier, x, (MIXED * 2)[:12], LENS, ids, q, 8)


def test_one_draft_refused_at_every_vocabulary_place(verifier):
    """A draft without a chance, the draw on each place of a small row."""
    V, R = 130, 130
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(2 * R, V, generator=gen)
    x[::2, 5] = float("-inf")
    ids = torch.full((R,), 5)
    q = torch.full((R, V), 1e-9)
    q[:, 5] = 1.0
    p = torch.softmax(x[::2].double(), 1).numpy()
    order = np.array([t if t != 5 else 4 for t in range(V)])
    cum = np.cumsum(np.maximum(p - q.double().numpy(), 0), 1)
    u = np.zeros(2 * R)
    u[::2] = 0.5
    for r in range(R):
        t = order[r]
        u[2 * r + 1] = ((cum[r, t - 1] if t else 0.0) + cum[r, t]) / (2 * cum[r, -1])
    plan = verifier.plan([SamplingParams(temperature=1.0)] * R, [1] * R, V)
    got = verifier.verify(plan, x.to(DEV), ids.to(DEV), torch.from_numpy(u).to(DEV), q.to(DEV))
    assert got.accepted.tolist() == [0] * R
    assert got.tokens[:, 0].tolist() == order.tolist()
    assert got.tokens[:, 1].tolist() == [-1] * R


def test_penalised_rows_count_their_drafts(verifier):
    V = 10000
    pen = [SamplingParams(temperature=0.9, repetition_penalty=1.3, frequency_penalty=0.4, presence_penalty=0.2),
           SamplingParams(repetition_penalty=1.5), SamplingParams(temperature=1.1, top_p=0.9, presence_penalty=1.0),
           SamplingParams(temperature=1.0)]
    lens = [4, 3, 5, 2]
    x, ids, q = make(21, 4, lens, V, torch.float16, True)
    rng = np.random.default_rng(5)
    contexts = [rng.integers(0, V, n).tolist() for n in (300, 0, 70, 10)]
    contexts[0] += ids[:4].tolist() * 3
    for probs in (q, None):
        check(verifier, x, pen, lens, ids, probs, 22, contexts)


@pytest.mark.parametrize("V, times", [(20001, 40), (70001, 12)])
@pytest.mark.parametrize("penalties", [False, True])
def test_large_batches_answer_as_small_ones(verifier, V, times, penalties):
    """The same requests many times over (another split of the rows over workgroups), the small
    batch checked against 64 bits."""
    params = [SamplingParams(temperature=1.0), SamplingParams(temperature=0.7, top_p=0.9)] * 6
    if penalties:
        params = [SamplingParams(temperature=p.temperature, top_p=p.top_p, presence_penalty=0.3, repetition_penalty=1.2)
                  for p in params]
    x, ids, q = make(V, 12, LENS, V, torch.bfloat16, True)
    rng = np.random.default_rng(V)
    contexts = [rng.integers(1, V, 200).tolist() for _ in range(12)] if penalties else None
    u, tokens, accepted, _ = plain(x.float().numpy(), params, LENS, ids.numpy(), q.numpy(), rng, contexts)
    drafts, at = [], 0
    for n in LENS:
        drafts.append(ids[at:at + n].tolist())
        at += n
    g = [x.to(DEV), ids.to(DEV), torch.from_numpy(u).to(DEV), q.to(DEV)]
    for n in (1, times):
        plan = verifier.plan(params * n, LENS * n, V, None if contexts is None else contexts * n, drafts * n)
        got = verifier.verify(plan, g[0].repeat(n, 1), g[1].repeat(n), g[2].repeat(n), g[3].repeat(n, 1))
        np.testing.assert_array_equal(got.accepted.cpu().numpy(), np.tile(accepted, n))
        np.testing.assert_array_equal(got.tokens.cpu().numpy(), np.tile(tokens, (n, 1)))


def test_longest_drafts(verifier):
    lens = [MAX_DRAFTS, 0, 200]
    x, ids, q = make(31, 3, lens, 300, torch.float32, True)
    # a draft model that is right nearly always: long runs of kept drafts
    last = np.zeros(sum(lens) + 3, bool)
    last[np.cumsum(np.array(lens) + 1) - 1] = True
    q = torch.softmax(x[torch.from_numpy(~last)], 1)
    _, accepted, _ = check(verifier, x, [SamplingParams(temperature=1.0)] * 3, lens, ids, q, 32)
    assert accepted.max() > 20


def test_odd_draft_values(verifier):
    """q below 0, NaN and infinite; ids outside the vocabulary; p never over q."""
    V = 5000
    lens = [1] * 8
    x, ids, q = make(41, 8, lens, V, torch.float32, True)
    q[0, :100] = -3.0
    q[1, 5:4000] = float("nan")
    q[2] = float("inf")
    q[3] = 2.0                           # nothing left: the row's most likely token
    q[4, :4990] = float("inf")
    ids[5], ids[6] = V, -1
    check(verifier, x, [SamplingParams(temperature=1.0)] * 8, lens, ids, q, 42)


def test_nothing_left_gives_the_first_of_equal_tokens(verifier):
    """p never over q on rows without filters, where the divide by the temperature makes two
    logits equal: the lower index, though its logit is the smaller."""
    V, s = 20000, np.float32(1.7)
    hi = np.float32(7.0)                 # 7 / 1.7 is past 4: its unit is hi's own
    for _ in range(100):
        if hi / s == np.nextafter(hi, np.float32(0)) / s:
            break
        hi = np.nextafter(hi, np.float32(8))
    assert hi / s == np.nextafter(hi, np.float32(0)) / s
    lo = np.nextafter(hi, np.float32(0))
    gen = torch.Generator().manual_seed(4)
    x = torch.randn(8, V, generator=gen)
    for r, (i, j) in enumerate([(12000, 300), (19999, 0), (0, 7), (9000, 8999)]):
        x[2 * r, i], x[2 * r, j] = float(hi), float(lo)
    q = torch.full((4, V), 2.0)
    pen = SamplingParams(temperature=1.7, presence_penalty=0.5)
    for params, ctx in (([SamplingParams(temperature=1.7)] * 4, None), ([pen] * 4, [[50, 51]] * 4)):
        plan = verifier.plan(params, [1] * 4, V, ctx, [[5]] * 4)
        got = verifier.verify(plan, x.to(DEV), torch.full((4,), 5, device=DEV), torch.full((8,), 0.6, dtype=torch.float64, device=DEV),
                              q.to(DEV))
        assert got.accepted.tolist() == [0] * 4
        assert got.tokens[:, 0].tolist() == [300, 0, 0, 8999]


def kept_drafts(x, lens):
    """Draft ids and certain-to-be-kept uniforms: the argmax of each drafted row, u = 0."""
    last = np.zeros(len(x), bool)
    last[np.cumsum(np.array(lens) + 1) - 1] = True
    return last, x.float().argmax(1)[torch.from_numpy(~last)]


@pytest.mark.parametrize("kind", ["peaked", "flat", "flatter", "grid", "equal", "two", "masked", "one", "steep", "tiles"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_draws_without_filters(verifier, kind, dtype):
    """Every draft kept, then the draw in rank order over the whole row: the canonical draw, bit
    for bit, at places all over the row, where the spans are counted side by side."""
    V, R = 70001, 24
    lens = [1, 0] * (R // 2)
    gen = torch.Generator().manual_seed(len(kind))
    x = torch.randn(sum(lens) + R, V, generator=gen)
    if kind == "peaked":
        x = 0.5 * x - 1.1 * torch.log(1.0 + torch.argsort(torch.rand(len(x), V, generator=gen), 1).float())
    elif kind == "flat":
        x = 0.3 * x
    elif kind == "flatter":
        x = 0.01 * x
    elif kind == "grid":
        x = torch.round(2.0 * x)
    elif kind == "equal":
        x = torch.full_like(x, -3.25)
    elif kind == "two":
        x = torch.where(x > 0.5, 1.0, 1.0 - 2.0 ** -6)
    elif kind == "masked":
        x[torch.rand(len(x), V, generator=gen) < 0.9] = float("-inf")
        x[::2, :40000] = torch.finfo(dtype).min
    elif kind == "one":
        x[:] = float("-inf")
        x[:, 51111] = 2.0
    elif kind == "steep":
        x = 12.0 * x
    elif kind == "tiles":                        # one tile far above the rest
        x[:, 4096:6144] += 25.0
    x = x.to(dtype)
    last, ids = kept_drafts(x, lens)
    params = [SamplingParams(temperature=t) for t in (1.0, 0.7, 1.7)] * (R // 3)
    rows = [p for p, n in zip(params, lens) for _ in range(n + 1)]
    u = np.zeros(len(rows))
    spots = np.concatenate([[0.0, 1.0 - 2.0 ** -53, 0.5, 1e-9, 1.0 - 1e-9], np.random.default_rng(5).random(R - 5)])
    u[last] = spots
    want = O.canonical_step(x.float().numpy(), O.resolve(rows, V), u)
    plan = verifier.plan(params, lens, V)
    assert plan.verify_args.draws == 1
    got = verifier.verify(plan, x.to(DEV), ids.to(DEV), torch.from_numpy(u).to(DEV))
    assert got.accepted.tolist() == lens
    drawn = got.tokens.gather(1, got.accepted.long()[:, None])[:, 0].cpu().numpy()
    np.testing.assert_array_equal(drawn, want.tokens[last])


def test_draws_without_filters_count_penalties(verifier):
    V, R = 80000, 20
    lens = [2, 0] * (R // 2)
    gen = torch.Generator().manual_seed(77)
    x = (0.5 * torch.randn(sum(lens) + R, V, generator=gen)).to(torch.bfloat16)
    rng = np.random.default_rng(6)
    contexts = [rng.integers(0, V, 3000).tolist() + [0] for _ in range(R)]
    pen = [SamplingParams(temperature=0.9, repetition_penalty=1.3, frequency_penalty=0.4)] * R
    last = np.zeros(len(x), bool)
    last[np.cumsum(np.array(lens) + 1) - 1] = True
    ids = torch.from_numpy(rng.integers(0, V, sum(lens)))
    u, tokens, accepted, _ = plain(x.float().numpy(), pen, lens, ids.numpy(), None, rng, contexts)
    plan = verifier.plan(pen, lens, V, contexts, [ids[2 * (i // 2):2 * (i // 2) + n].tolist() for i, n in enumerate(lens)])
    assert plan.verify_args.draws == 1
    got = verifier.verify(plan, x.to(DEV), ids.to(DEV), torch.from_numpy(u).to(DEV))
    np.testing.assert_array_equal(got.accepted.cpu().numpy(), accepted)
    np.testing.assert_array_equal(got.tokens.cpu().numpy(), tokens)


def test_a_draw_past_the_candidates_at_a_middle_key(verifier):
    """Many tokens of a few keys in one part of one bin: the search over the keys."""
    V, R = 66000, 20
    x = torch.zeros(R, V)
    base = torch.tensor(5.0)
    for i in range(6):                                    # six neighbouring fp32 values
        x[:, i::6] = base
        base = torch.nextafter(base, torch.tensor(0.0))
    u = np.random.default_rng(8).random(R)
    params = [SamplingParams(temperature=1.0)] * R
    want = O.canonical_step(x.numpy(), O.resolve(params, V), u)
    plan = verifier.plan(params, [0] * R, V)
    got = verifier.verify(plan, x.to(DEV), torch.zeros(0, dtype=torch.int64, device=DEV), torch.from_numpy(u).to(DEV))
    np.testing.assert_array_equal(got.tokens[:, 0].cpu().numpy(), want.tokens)


def test_strides_and_alignment(verifier):
    V = 4099
    x, ids, q = make(51, 12, LENS, V, torch.bfloat16, True)

    def spread(g):
        big = torch.full((g[0].shape[0], V + 13), float("nan"), dtype=g[0].dtype, device=DEV)
        big[:, 5:5 + V] = g[0]
        wide = torch.full((g[3].shape[0], V + 3), float("nan"), device=DEV)
        wide[:, 1:1 + V] = g[3]
        ids2 = torch.stack([g[1], g[1] * 0 - 7], 1)[:, 0]
        return [big[:, 5:5 + V], ids2, torch.stack([g[2], g[2] * 0 - 7], 1)[:, 0], wide[:, 1:1 + V]]

    params = (MIXED * 2)[:12]
    check(verifier, x, params, LENS, ids, q, 52, transform=spread)
    check(verifier, x, params, LENS, ids, q, 52,
          transform=lambda g: [g[0].t().contiguous().t(), g[1], g[2], g[3].t().contiguous().t()])


def test_another_stream_and_a_reused_plan(verifier):
    V = 3000
    params = (MIXED * 2)[:12]
    x, ids, q = make(61, 12, LENS, V, torch.float32, True)
    _, _, want = check(verifier, x, params, LENS, ids, q, 62)
    u, tokens, _, _ = plain(x.float().numpy(), params, LENS, ids.numpy(), q.numpy(), np.random.default_rng(62))
    plan = verifier.plan(params, LENS, V)
    g = [x.to(DEV), ids.to(DEV), torch.from_numpy(u).to(DEV), q.to(DEV)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            got = verifier.verify(plan, *g)
            np.testing.assert_array_equal(got.tokens.cpu().numpy(), want)
    torch.cuda.current_stream().wait_stream(side)


def test_a_plan_made_on_a_busy_stream(verifier):
    V = 3000
    params = (MIXED * 2)[:12]
    x, ids, q = make(63, 12, LENS, V, torch.float32, True)
    u, want, _, _ = plain(x.float().numpy(), params, LENS, ids.numpy(), q.numpy(), np.random.default_rng(64))
    g = [x.to(DEV), ids.to(DEV), torch.from_numpy(u).to(DEV), q.to(DEV)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)           # some 20 ms in front of the settings' upload
        plan = verifier.plan(params, LENS, V)
    got = verifier.verify(plan, *g)
    del plan
    np.testing.assert_array_equal(got.tokens.cpu().numpy(), want)


def test_graph_replay(verifier):
    V = 20000
    params = (MIXED * 2)[:12]
    x, ids, q = make(71, 12, LENS, V, torch.bfloat16, True)
    plan = verifier.plan(params, LENS, V)
    rng = np.random.default_rng(0)
    g = [x.to(DEV), ids.to(DEV), torch.from_numpy(rng.random(plan.rows)).to(DEV), q.to(DEV)]
    verifier.verify(plan, *g)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = verifier.verify(plan, *g)
    for _ in range(4):
        g[2].copy_(torch.from_numpy(rng.random(plan.rows)))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in got]
        eager = verifier.verify(plan, *g)
        for a, b in zip(replayed, eager):
            assert torch.equal(a, b)


def test_emitted_tokens_follow_the_target(verifier):
    """The first token's distribution is the target's whatever the draft's: 40000 requests of
    one draft on 6 tokens.  Each count is binomial; 5 standard deviations."""
    R, V = 40000, 6
    gen = torch.Generator(device=DEV).manual_seed(9)
    x = torch.tensor([1.0, 0.0, -1.0, 2.0, 0.5, -2.0], device=DEV).expand(2 * R, V).contiguous()
    p = torch.softmax(x[0].double(), 0)
    q = torch.tensor([0.3, 0.3, 0.2, 0.05, 0.05, 0.1], device=DEV).expand(R, V).contiguous()
    ids = torch.multinomial(q, 1, generator=gen)[:, 0]
    u = torch.rand(2 * R, dtype=torch.float64, generator=gen, device=DEV)
    plan = verifier.plan([SamplingParams(temperature=1.0)] * R, [1] * R, V)
    got = verifier.verify(plan, x, ids, u, q)
    counts = torch.bincount(got.tokens[:, 0], minlength=V).double()
    assert ((counts - R * p).abs() <= 5 * (R * p * (1 - p)).sqrt()).all(), counts


def test_device_draws_equal_the_uniforms_they_stand_for(verifier):
    V = 3000
    params = (MIXED * 2)[:12]
    x, ids, q = make(81, 12, LENS, V, torch.float32, True)
    rows = sum(LENS) + 12
    rng = np.random.default_rng(3).integers(0, 2 ** 63, (rows, 3)).astype(np.uint64)
    u = verifier._fused.uniforms(torch.from_numpy(rng.view(np.int64)).to(DEV))
    g = [x.to(DEV), ids.to(DEV)]
    a = verifier.verify(verifier.plan(params, LENS, V, rng=rng), *g, None, q.to(DEV))
    b = verifier.verify(verifier.plan(params, LENS, V), *g, u, q.to(DEV))
    for s, t in zip(a, b):
        assert torch.equal(s, t)


def test_offsets_that_do_not_fit_are_answered_without_tokens(verifier):
    V = 64
    x = torch.randn(6, V, device=DEV)
    plan = verifier.plan([SamplingParams(temperature=1.0)] * 3, [1, 1, 1], V)
    plan._offsets.copy_(torch.tensor([0, 2, 1, 9]))          # 2 > max_drafts, below 0 drafts, past the end
    got = verifier.verify(plan, x, torch.zeros(3, dtype=torch.int64, device=DEV),
                          torch.rand(6, dtype=torch.float64, device=DEV))
    assert got.accepted.tolist() == [-1, -1, -1]
    assert (got.tokens == -1).all()


def test_refusals(verifier):
    V = 64
    plan = verifier.plan([SamplingParams(temperature=1.0)] * 2, [1, 2], V)
    x = torch.randn(5, V, device=DEV)
    ids = torch.zeros(3, dtype=torch.int64, device=DEV)
    u = torch.rand(5, dtype=torch.float64, device=DEV)
    q = torch.rand(3, V, device=DEV)
    for bad in ([x[:4], ids, u, q], [x[:, :63], ids, u, q], [x, ids[:2], u, q], [x, ids.int(), u, q], [x, ids, u[:4], q],
                [x, ids, u.float(), q], [x, ids, None, q], [x, ids, u, q[:2]], [x, ids, u, q.double()],
                [x.cpu(), ids, u, q], [x, ids.cpu(), u, q], [x, ids, u, q.cpu()]):
        with pytest.raises(ValueError):
            verifier.verify(plan, *bad)
    one = [SamplingParams(temperature=1.0)]
    for args in ((one, [1, 2], V), (one, [-1], V), (one, [MAX_DRAFTS + 1], V), (one, [1], 0),
                 (one, [1], _lib.MAX_VOCAB + 1), ([SamplingParams(logprobs=1)], [1], V),
                 ([SamplingParams(presence_penalty=1.0)], [1], V, [[1]]), (one, [1], V, None, [[1, 2]])):
        with pytest.raises(ValueError):
            verifier.plan(*args)
    none = verifier.verify(verifier.plan([], [], V), x[:0], ids[:0], u[:0])
    assert none.tokens.shape == (0, 1)


@pytest.mark.parametrize("V", [300, 70001])
def test_rows_of_nothing(verifier, V):
    """Rows of -inf alone, among ordinary ones: the first token, whatever the settings."""
    lens = [1, 0, 2, 1] * 6
    x, ids, q = make(V, 24, lens, V, torch.float32, True)
    x[::2] = float("-inf")
    x[-3:] = float("-inf")
    for probs in (q, None):
        check(verifier, x, (MIXED * 4), lens, ids, probs, 5)


def test_large_offsets(verifier):
    """Rows of logits and draft probabilities 2^31 elements apart."""
    V, step = 1000, 2 ** 31 + 8
    x, ids, q = make(91, 1, [1], V, torch.float16, True)
    far = [torch.empty(step + V, dtype=torch.float16, device=DEV) for _ in range(2)]

    def spread(g):
        a = torch.as_strided(far[0], (2, V), (step, 1))
        a.copy_(g[0])
        b = torch.as_strided(far[1], (2, V), (step, 1))
        b[1].copy_(g[3][0])
        b[0].copy_(g[3][0])
        return [a, g[1], g[2], b[1:2]]

    check(verifier, x, [SamplingParams(temperature=1.0)], [1], ids, q.half(), 92, transform=spread)
