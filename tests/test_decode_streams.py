"""Memory that a bank, a search or a pool of pages keeps is marked for every stream that uses it, so it is not
handed out while that stream's kernels are on their way: the bookkeeping on the CPU with stand-ins for streams
and launches, and answers on an MI355X."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from fie_amd import adapters, beam, pages
from fie_amd.adapters import AdapterBank, adapter_linear
from fie_amd.beam import BeamSearch, Beams, first_beams
from fie_amd.pages import CachePages


class OnDevice(torch.Tensor):
    """A host tensor that says it is on device 0, and keeps which streams it was marked for."""

    def get_device(self):
        return 0

    def record_stream(self, stream):
        self.__dict__.setdefault("used_on", []).append(stream)


def used(*tensors):
    return [t.__dict__.get("used_on", []) for t in tensors]


@pytest.fixture
def machine(monkeypatch):
    """[the current stream, whether it captures, launches]"""
    m = SimpleNamespace(stream=0, capturing=False, launches=0)

    def run(*args):
        m.launches += 1

    for module in (adapters, beam, pages):
        monkeypatch.setattr(module, "_raw_stream", lambda index: m.stream, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: m.stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: m.stream)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: m.capturing)
    monkeypatch.setattr(adapters, "_run", run)
    monkeypatch.setattr(adapters, "_size", lambda args: 64)
    monkeypatch.setattr(beam, "_run", run)
    monkeypatch.setattr(beam, "_size", lambda args: 64)
    monkeypatch.setattr(pages, "_launch", run)
    return m


def on_device(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype).as_subclass(OnDevice)


def test_a_bank_on_another_stream(machine):
    bank = AdapterBank.__new__(AdapterBank)
    bank.adapters, bank.k, bank.n, bank.rank, bank.rank_pad, bank.k_pad, bank.b_pitch = 2, 4, 6, 3, 16, 64, 16
    bank.dtype, bank.index, bank._made_on = torch.float32, 0, 0
    bank.a, bank.b, bank.scale, bank.ranks = on_device(2, 16, 64), on_device(2, 6, 16), on_device(2), on_device(2, dtype=torch.int32)
    own = bank.a, bank.b, bank.scale, bank.ranks
    plan = SimpleNamespace(tokens=5, adapters=2, index=0, data=on_device(9, dtype=torch.int32), on_stream=lambda: None)
    x = on_device(5, 4)
    adapter_linear(x, bank, plan)
    assert used(*own) == [[]] * 4
    machine.stream = 7
    adapter_linear(x, bank, plan)
    assert used(*own) == [[7]] * 4
    machine.capturing = True
    adapter_linear(x, bank, plan)
    assert used(*own) == [[7]] * 4 and machine.launches == 3
    machine.capturing, machine.stream = False, 8
    bank.load(1, on_device(3, 4), on_device(6, 3))
    assert used(*own) == [[7, 8]] * 4


def test_a_search_on_another_stream(machine):
    search = BeamSearch.__new__(BeamSearch)
    search.requests, search.count, search.max_tokens, search.device, search._made_on, search._index = 2, 3, 4, torch.device("cpu"), 0, 0
    search._settings = dict(eos=(1,), length_penalty=1.0, early_stopping=False, min_tokens=0, max_tokens=4, pad=0)
    search.beams = Beams(*(t.as_subclass(OnDevice) for t in first_beams(2, 3, "cpu")))
    search._history = on_device(4, 6, dtype=torch.int32), on_device(4, 6, dtype=torch.int32)
    own = *search.beams, *search._history
    x = on_device(6, 10)
    search.step(x)
    assert used(*own) == [[]] * 7
    machine.stream = 7
    search.step(x)
    assert used(*own) == [[7]] * 7
    machine.capturing = True
    search.step(x)
    assert used(*own) == [[7]] * 7 and machine.launches == 3
    machine.capturing, machine.stream = False, 8
    search.stop([1])
    assert used(*own) == [[7, 8]] * 7
    search.restart([0])
    assert used(*own) == [[7, 8, 8]] * 7


def test_caches_added_on_another_stream_than_the_pools(machine):
    pool = CachePages.__new__(CachePages)
    pool.pages, pool.page_size, pool.rows, pool.max_pages, pool.device, pool._index = 8, 4, 2, 3, torch.device("cpu"), 0
    pool.state, pool._scratch, pool._groups, pool._made_on = on_device(30, dtype=torch.int32), on_device(64), [], 0
    cache = on_device(8, 4, 2)

    def add():
        pool.add_caches([cache])
        layout, tensors, base = pool._groups.pop()
        pool._groups.append((layout, tensors, base.as_subclass(OnDevice)))
        return pool._groups[-1][2]

    first = add()
    pool.step(None)
    assert used(first, pool.state, pool._scratch) == [[]] * 3
    machine.stream = 7
    second = add()
    machine.stream = 0                                  # the pool's own, not the second addresses'
    pool.step(None)
    assert used(second) == [[0]]
    machine.stream = 9
    pool.compact()
    assert [u[-1] for u in used(first, second, pool.state, pool._scratch)] == [9] * 4


DEV = "cuda:0"


@pytest.mark.gpu
def test_a_bank_and_a_search_dropped_on_a_side_stream():
    gen = torch.Generator(device=DEV).manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731

    def bank():
        got = AdapterBank(4, 512, 640, 16, torch.bfloat16, DEV)
        g = torch.Generator(device=DEV).manual_seed(2)
        for i in range(4):
            got.load(i, torch.randn(16, 512, generator=g, device=DEV) / 20, torch.randn(640, 16, generator=g, device=DEV))
        return got

    x, logits = rnd(300, 512).bfloat16(), [rnd(32, 5000) for _ in range(3)]
    ids = torch.randint(0, 4, (300,), generator=gen, device=DEV, dtype=torch.int32)
    keep = bank()
    want = adapter_linear(x, keep, keep.plan(ids))
    search = BeamSearch(DEV, 8, 4, max_tokens=9)
    wanted = [search.step(v).tokens for v in logits]
    mine, search = bank(), BeamSearch(DEV, 8, 4, max_tokens=9)
    sizes = [t.numel() * t.element_size() for t in (mine.a, mine.b, mine.scale, mine.ranks, *search.beams, *search._history)]
    plan = mine.plan(ids)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        got = adapter_linear(x, mine, plan)
        chosen = [search.step(v).tokens for v in logits]
    del mine, search
    junk = [torch.full((n,), 0xFF, dtype=torch.uint8, device=DEV) for n in sizes for _ in range(4)]
    side.synchronize()
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(chosen, wanted))
    assert all(int(j.min()) == 0xFF for j in junk)
