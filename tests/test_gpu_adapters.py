"""Low-rank adapters on an MI355X against 64 bits.

h = A x is a sum of k exact products in fp32: off by k * 2^-24 of the sum of their magnitudes at most
(and 40 more for the partial sums).  Two-byte adapters take it as two numbers: 2^-8 * 2^-8 of |h|
off in bf16, 2^-11 * 2^-11 in fp16 and, of a row whose largest |h| is m, the trailing part's last
bit, 2^-24 m.  The second product adds 2 * rank terms in fp32, the scale and the base a rounding each;
then half a unit of the output's type.
"""

from __future__ import annotations

import random

import pytest
import torch

from fie_amd.adapters import AdapterBank, adapter_linear
from fie_amd.linear import int8_linear, quantize_rows
from fie_amd.norm import block_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
UNIT = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def make(seed, adapters, k, n, rank, dtype, ranks=None):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    bank = AdapterBank(adapters, k, n, rank, dtype, DEV)
    pairs = []
    for i in range(adapters):
        r = ranks[i] if ranks is not None else max(0, rank - (i % 4) * (rank // 3))
        a, b, s = (rnd(r, k) / k ** 0.5).to(dtype), rnd(n, r).to(dtype), 0.5 + 0.25 * (i % 3)
        bank.load(i, a, b, s)
        pairs.append((a.double(), b.double(), s))
    return bank, pairs, rnd


def check(got, x, pairs, ids, base=None, half=None):
    x = x.double()
    dtype = got.dtype
    t, n = x.shape[0], got.shape[-1]
    split = {torch.float32: 0.0, torch.float16: 2.0 ** -22, torch.bfloat16: 2.0 ** -16}[half]
    b0 = torch.zeros(t, n, dtype=torch.float64, device=DEV) if base is None else base.double().reshape(t, n)
    want, off = b0.clone(), torch.zeros_like(b0)
    for i, (a, b, s) in enumerate(pairs):
        at = (ids == i).nonzero()[:, 0]
        if not len(at) or not a.shape[0]:
            continue
        h, size = x[at] @ a.T, x[at].abs() @ a.abs().T
        want[at] += s * (h @ b.T)
        h_off = UNIT * (x.shape[1] + 40) * size + split * h.abs()
        if half == torch.float16:
            h_off = h_off + UNIT * h.abs().amax(1, keepdim=True)
        off[at] += abs(s) * (h_off @ b.abs().T + UNIT * (2 * a.shape[0] + 4) * (h.abs() @ b.abs().T))
    off = off + 2 * UNIT * (b0.abs() + (want - b0).abs())
    bound = off + HALF[dtype] * (want.abs() + off) * 1.01 + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    mine = got.double().reshape(t, n)
    bad = torch.where(want.isnan(), ~mine.isnan(), ~((mine - want).abs() <= bound))     # infinities' sums are no numbers
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), got.reshape(t, n)[bad][:4].tolist(), want[bad][:4].tolist())


def some_ids(seed, tokens, adapters, runs=1, none=0.2):
    rng = random.Random(seed)
    ids = []
    while len(ids) < tokens:
        ids += [-1 if rng.random() < none else rng.randrange(adapters)] * rng.randint(1, runs)
    return torch.tensor(ids[:tokens], dtype=torch.int32, device=DEV)


SIZES = [(1, 1, 1, 1, 1), (1, 1, 64, 16, 1), (1, 8, 4096, 4096, 16), (2, 3, 31, 7, 3), (5, 2, 127, 33, 16), (16, 1, 128, 256, 8),
         (17, 3, 129, 257, 17), (33, 40, 1000, 500, 16), (64, 5, 2048, 1023, 32), (77, 33, 1003, 5001, 24), (250, 64, 1024, 2048, 16),
         (300, 7, 333, 1111, 33), (513, 2, 4097, 640, 64), (700, 3, 256, 300, 100), (1500, 5, 640, 777, 48), (1024, 4, 515, 258, 256),
         (40, 4096, 70, 50, 4)]


@pytest.mark.parametrize("tokens, adapters, k, n, rank", SIZES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_sizes(tokens, adapters, k, n, rank, dtype):
    print(f"  case: {tokens} of {adapters}, {k} to {n}, rank {rank} {dtype}", flush=True)
    bank, pairs, rnd = make(tokens + k, adapters, k, n, rank, dtype)
    x = rnd(tokens, k).to(dtype)
    for runs in (1, 100):
        ids = some_ids(k + runs, tokens, adapters, runs)
        plan, base = bank.plan(ids), rnd(tokens, n)
        check(adapter_linear(x, bank, plan, base=base.to(dtype)), x, pairs, ids, base.to(dtype), half=dtype)
        check(adapter_linear(x, bank, plan, base=base), x, pairs, ids, base, half=dtype)
        check(adapter_linear(x, bank, plan, out_dtype=torch.float32), x, pairs, ids, half=dtype)
        q, scale = quantize_rows(x)
        got = adapter_linear(q, bank, plan, x_scale=scale, base=base)
        check(got, q.double() * scale.double()[:, None], pairs, ids, base, half=dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_without_adapters_keep_their_base(dtype):
    bank, pairs, rnd = make(1, 4, 100, 130, 8, dtype, ranks=[8, 0, 3, 8])
    x, base = rnd(50, 100).to(dtype), rnd(50, 130).to(dtype)
    for ids in ([-1] * 50, [1] * 50, [-5, 4, 2 ** 31 - 1, -2 ** 31, 1] * 10, [0, -1, 1, 2, 3] * 10):
        ids = torch.tensor(ids, dtype=torch.int32, device=DEV)
        plan = bank.plan(ids)
        got = adapter_linear(x, bank, plan, base=base)
        keep = (ids < 0) | (ids > 3) | (ids == 1)
        assert torch.equal(got[keep], base[keep])
        check(got, x, pairs, ids, base, half=dtype)
        assert (adapter_linear(x, bank, plan)[keep] == 0).all()
        mine = base.clone()
        assert adapter_linear(x, bank, plan, base=mine, out=mine) is mine and torch.equal(mine, got)
    # a token's NaN is its own, and other adapters' are no one else's
    x[3] = float("nan")
    bank.load(2, torch.full((3, 100), float("nan")), torch.full((130, 3), float("inf")), 1.0)
    ids = torch.tensor([0, 3, -1, 0, 2] * 10, dtype=torch.int32, device=DEV)
    got = adapter_linear(x, bank, bank.plan(ids), base=base)
    bad = (ids == 2)
    bad[3] = True
    assert got[bad].isnan().all() and torch.isfinite(got[~bad]).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_wide_ranges(dtype):
    """h past fp16's largest, and far below its least."""
    bank, pairs, rnd = make(2, 1, 512, 64, 16, dtype)
    ids = torch.zeros(8, dtype=torch.int32, device=DEV)
    x = rnd(8, 512)
    x *= torch.tensor([1e4, 1e3, 1.0, 1e-3, 1e-4, 1e-5, 3e4, 0.0], device=DEV)[:, None]
    x = x.to(dtype)
    a, b, _ = pairs[0]
    bank.load(0, 8.0 * a, 2.0 ** -10 * b, 1.0)
    got = adapter_linear(x, bank, bank.plan(ids), out_dtype=torch.float32)
    check(got, x, [((8.0 * a).to(dtype).double(), (2.0 ** -10 * b).to(dtype).double(), 1.0)], ids, half=dtype)
    h = x.double() @ (8.0 * a).T
    assert float(h[torch.isfinite(h)].abs().max()) > 65504.0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("at, pad", [(0, 0), (1, 0), (1, 2), (2, 6), (4, 4), (3, 5), (8, 8)])
def test_strides_and_alignment(at, pad, dtype):
    for tokens, k, n in ((20, 200, 130), (600, 136, 260)):
        bank, pairs, rnd = make(3, 3, k, n, 20, dtype)
        ids = some_ids(5, tokens, 3, 50)

        def wide(t, fill=7.0):
            room = torch.full((t.shape[0], at + t.shape[1] + pad), fill, device=DEV).to(t.dtype)
            room[:, at:at + t.shape[1]] = t
            return room, room[:, at:at + t.shape[1]]

        x, base = rnd(tokens, k).to(dtype), rnd(tokens, n).to(dtype)
        plan = bank.plan(ids)
        want = adapter_linear(x, bank, plan, base=base)
        check(want, x, pairs, ids, base, half=dtype)
        out, y = wide(torch.zeros_like(base))
        got = adapter_linear(wide(x, float("nan"))[1], bank, plan, base=wide(base)[1], out=y)
        assert got is y and torch.equal(y, want)
        assert (out[:, :at] == 7).all() and (out[:, at + n:] == 7).all()
        q, s = quantize_rows(x)
        other = adapter_linear(q, bank, plan, x_scale=s, base=base)
        assert torch.equal(adapter_linear(wide(q, 99)[1], bank, plan, x_scale=s, base=wide(base)[1]), other)
    assert torch.equal(adapter_linear(x.t().contiguous().t(), bank, plan, base=base.t().contiguous().t()), want)
    assert torch.equal(adapter_linear(x.view(2, 300, k), bank, plan, base=base.view(2, 300, n)).view(600, n), want)
    one = x[:1].expand(600, k)
    check(adapter_linear(one, bank, plan, base=base[:1].expand(600, n)), one, pairs, ids, base[:1].expand(600, n), half=dtype)


@pytest.mark.parametrize("tokens", [1, 15, 16, 17, 63, 64, 65, 511, 512, 513, 2000])
def test_tiles_of_one_adapter(tokens):
    for adapters in (1, 200):
        bank, pairs, rnd = make(tokens, adapters, 96, 80, 16, torch.bfloat16)
        x = rnd(tokens, 96).bfloat16()
        for ids in (torch.zeros(tokens, dtype=torch.int32, device=DEV), some_ids(1, tokens, adapters, 3)):
            check(adapter_linear(x, bank, bank.plan(ids)), x, pairs, ids, half=torch.bfloat16)


def test_past_32_bit_offsets():
    """Outputs of more than 2^31 elements, and banks of more than 2^31 bytes."""
    tokens, k, n = 70000, 64, 32768
    bank, pairs, rnd = make(4, 2, k, n, 4, torch.bfloat16)
    ids = torch.full((tokens,), -1, dtype=torch.int32, device=DEV)
    ids[[0, 1, 40000, tokens - 2, tokens - 1]] = torch.tensor([0, 1, 0, 1, 0], dtype=torch.int32, device=DEV)
    x = rnd(tokens, k).bfloat16()
    got = adapter_linear(x, bank, bank.plan(ids))
    some = torch.tensor([0, 1, 40000, tokens - 2, tokens - 1], device=DEV)
    check(got[some], x[some], pairs, ids[some], half=torch.bfloat16)
    assert int(got.count_nonzero(1).gt(0).sum()) == 5
    del got
    bank, pairs, rnd = make(5, 300, 4096, 131072, 16, torch.bfloat16, ranks=[16 if i in (0, 299) else 0 for i in range(300)])
    ids = torch.tensor([299, 0, 1], dtype=torch.int32, device=DEV)
    x = rnd(3, 4096).bfloat16()
    check(adapter_linear(x, bank, bank.plan(ids)), x, pairs, ids, half=torch.bfloat16)


def test_beside_the_shared_product():
    """The end of a block with adapters: norm to int8, the shared product, the adapters on the same tokens."""
    T, H, N = 60, 1024, 2048
    bank, pairs, rnd = make(6, 5, H, N, 16, torch.bfloat16)
    w, ws = quantize_rows(rnd(N, H) / H ** 0.5)
    ids = some_ids(7, T, 5)
    plan = bank.plan(ids)
    normed = block_norm(rnd(T, H).bfloat16(), rnd(T, H).bfloat16(), quantize=True)
    base = int8_linear(normed.y, w, ws, x_scale=normed.scale, out_dtype=torch.float32)
    y = adapter_linear(normed.y, bank, plan, x_scale=normed.scale, base=base)
    assert y.dtype == torch.bfloat16
    check(y, normed.y.double() * normed.scale.double()[:, None], pairs, ids, base, half=torch.bfloat16)


def test_repeats_and_order_do_not_matter():
    bank, _, rnd = make(8, 9, 700, 900, 32, torch.bfloat16)
    x, base, ids = rnd(900, 700).bfloat16(), rnd(900, 900), some_ids(9, 900, 9)
    first = adapter_linear(x, bank, bank.plan(ids), base=base)
    for seed in range(4):
        order = torch.randperm(900, generator=torch.Generator().manual_seed(seed)).to(DEV)
        got = adapter_linear(x[order], bank, bank.plan(ids[order]), base=base[order])
        assert torch.equal(got, first[order])


def test_captured_with_its_plan():
    bank, _, rnd = make(10, 6, 512, 640, 16, torch.float16)
    x, base, ids = rnd(40, 512).half(), rnd(40, 640).half(), some_ids(1, 40, 6)
    adapter_linear(x, bank, bank.plan(ids), base=base)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = bank.plan(ids)
        got = adapter_linear(x, bank, plan, base=base)
        again = adapter_linear(x, bank, plan, base=got)
    for i in range(4):
        x.copy_(rnd(40, 512))
        base.copy_(rnd(40, 640))
        ids.copy_(some_ids(20 + i, 40, 6))
        graph.replay()
        torch.cuda.synchronize()
        plan2 = bank.plan(ids)
        want = adapter_linear(x, bank, plan2, base=base)
        assert torch.equal(got, want) and torch.equal(again, adapter_linear(x, bank, plan2, base=want))


def test_on_a_side_stream():
    bank, _, rnd = make(11, 6, 512, 640, 16, torch.bfloat16)
    x, base, ids = rnd(3000, 512).bfloat16(), rnd(3000, 640), some_ids(1, 3000, 6, 9)
    plan = bank.plan(ids)
    want = adapter_linear(x, bank, plan, base=base)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    size = plan.data.numel()
    with torch.cuda.stream(side):
        torch.cuda._sleep(10_000_000)
        got = adapter_linear(x, bank, plan, base=base)
    del plan
    junk = [torch.full((size,), 2 ** 31 - 1, dtype=torch.int32, device=DEV) for _ in range(6)]
    side.synchronize()
    assert torch.equal(got, want) and all(int(j.min()) == 2 ** 31 - 1 for j in junk)


def test_refusals():
    bank, _, rnd = make(12, 2, 64, 48, 8, torch.bfloat16)
    ids = torch.zeros(5, dtype=torch.int32, device=DEV)
    plan, x = bank.plan(ids), rnd(5, 64).bfloat16()
    q, s = quantize_rows(x)
    other = AdapterBank(3, 64, 48, 8, torch.bfloat16, DEV)
    y = torch.zeros(5, 48, dtype=torch.bfloat16, device=DEV)
    for call in (lambda: adapter_linear(x[:4], bank, plan), lambda: adapter_linear(x[:, :63], bank, plan),
                 lambda: adapter_linear(x.float(), bank, plan), lambda: adapter_linear(x.cpu(), bank, plan), lambda: adapter_linear(q, bank, plan),
                 lambda: adapter_linear(x, bank, plan, x_scale=s), lambda: adapter_linear(q, bank, plan, x_scale=s[:4]),
                 lambda: adapter_linear(q, bank, plan, x_scale=s.double()), lambda: adapter_linear(x, other, plan),
                 lambda: adapter_linear(x, bank, plan, out_dtype=torch.float16), lambda: adapter_linear(x, bank, plan, base=y[:4]),
                 lambda: adapter_linear(x, bank, plan, base=y.half()), lambda: adapter_linear(x, bank, plan, out=y[:, :40]),
                 lambda: adapter_linear(x, bank, plan, out=y, out_dtype=torch.float32), lambda: adapter_linear(x, bank, plan, out=y.cpu()),
                 lambda: adapter_linear(x, bank, plan, out=torch.zeros(48, 5, dtype=torch.bfloat16, device=DEV).t()),
                 lambda: adapter_linear(x, bank, plan, out=y[0].expand(5, 48)), lambda: bank.plan(ids.long()), lambda: bank.plan(ids.cpu()),
                 lambda: bank.plan(ids[None]), lambda: bank.load(2, rnd(8, 64), rnd(48, 8)), lambda: bank.load(-1, rnd(8, 64), rnd(48, 8)),
                 lambda: bank.load(0, rnd(9, 64), rnd(48, 9)), lambda: bank.load(0, rnd(8, 63), rnd(48, 8)),
                 lambda: bank.load(0, rnd(8, 64), rnd(48, 7)), lambda: AdapterBank(1, 64, 48, 257, torch.bfloat16, DEV),
                 lambda: AdapterBank(1, 64, 48, 8, torch.float64, DEV)):
        with pytest.raises(ValueError):
            call()
    empty = bank.plan(ids[:0])
    assert adapter_linear(x[:0], bank, empty).shape == (0, 48)
