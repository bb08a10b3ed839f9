"""A workspace's memory is not handed out while another stream's kernels use it: the bookkeeping
on the CPU with stand-ins for the allocator and the streams, and answers on an MI355X."""

from __future__ import annotations

import pytest
import torch

from fie_amd import kernel
from fie_amd.kernel import HELP_ROWS, FusedSampler
from fie_amd.runtime.sampling import SamplingParams
from fie_amd.verify import DraftVerifier


class Block:
    """A tensor on device 0, allocated on whatever stream was current."""

    device = torch.device("cuda:0")

    def __init__(self, address):
        self.address, self.used_on = address, []

    def data_ptr(self):
        return self.address

    def get_device(self):
        return 0

    def record_stream(self, stream):
        self.used_on.append(stream)


@pytest.fixture
def machine(monkeypatch):
    """[the current stream, whether it captures, the blocks allocated]"""
    m = dict(stream=0, capturing=False, blocks=[])

    def empty(n, **kw):
        m["blocks"].append(Block(256 * (1 + len(m["blocks"]))))
        return m["blocks"][-1]

    monkeypatch.setattr(kernel.torch, "empty", empty)
    monkeypatch.setattr(kernel, "_raw_stream", lambda index: m["stream"], raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: m["stream"])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: m["capturing"])
    return m


@pytest.mark.parametrize("rows", [4, 64])
def test_a_workspace_on_another_stream_is_marked(machine, rows):
    fs = FusedSampler("cuda:0")
    fs.ensure_workspace(rows, 1000)
    fs.ensure_workspace(rows, 900)
    first = machine["blocks"][0]
    assert first.used_on == []                              # its own stream
    machine["stream"] = 7
    fs.ensure_workspace(rows, 1000)
    assert first.used_on == [7]
    machine["capturing"] = True
    fs.ensure_workspace(rows, 1000)
    assert first.used_on == [7] and len(machine["blocks"]) == 1
    machine["capturing"] = False
    fs.ensure_workspace(rows, 2000)                         # grows on stream 7: that one's own from now on
    fs.ensure_workspace(rows, 2000)
    second = machine["blocks"][1]
    assert second.used_on == [] and len(machine["blocks"]) == 2
    machine["stream"] = 0
    fs.ensure_workspace(rows, 10)
    assert second.used_on == [0] and first.used_on == [7]


def test_small_and_large_batches_keep_their_own(machine):
    fs = FusedSampler("cuda:0")
    fs.ensure_workspace(HELP_ROWS, 1000)
    machine["stream"] = 5
    fs.ensure_workspace(HELP_ROWS + 1, 1000)
    fs.ensure_workspace(HELP_ROWS + 1, 1000)
    small, large = machine["blocks"]
    assert small.used_on == [] and large.used_on == []
    fs.ensure_workspace(1, 1000)
    assert small.used_on == [5]


@pytest.mark.gpu
def test_answers_while_the_workspace_moves_and_grows():
    """Verifications queued on a side stream, the workspace made on the main one, replaced and
    dropped while they are on their way, and the main stream filling whatever memory it gets."""
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev).manual_seed(1)
    params, lens = [SamplingParams(temperature=1.0), SamplingParams(temperature=0.8, top_p=0.9)] * 12, [2, 1] * 12
    sizes = (3000, 20001, 40000)
    rows, drafts = sum(lens) + 24, sum(lens)
    inputs = [(torch.randn(rows, V, generator=gen, device=dev), torch.randint(0, V, (drafts,), generator=gen, device=dev),
               torch.rand(rows, dtype=torch.float64, generator=gen, device=dev)) for V in sizes]
    ref = DraftVerifier(dev)
    want = [ref.verify(ref.plan(params, lens, V), *g) for V, g in zip(sizes, inputs)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    v = DraftVerifier(dev)
    v.verify(v.plan(params, lens, sizes[0]), *inputs[0])    # the workspace is the main stream's
    nbytes = v._fused._wss[False][0].numel()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        plans = [v.plan(params, lens, V) for V in sizes]
        torch.cuda._sleep(20_000_000)
        got = [v.verify(p, *g) for p, g in zip(plans, inputs)]
    del v
    junk = [torch.full((nbytes,), 0xFF, dtype=torch.uint8, device=dev) for _ in range(8)]
    side.synchronize()
    for a, b in zip(got, want):
        for s, t in zip(a, b):
            assert torch.equal(s, t)
    assert all(int(j.min()) == 0xFF for j in junk)
