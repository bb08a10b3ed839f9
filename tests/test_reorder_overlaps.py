"""Outputs of reorder_states that share memory with any state or output of the call are refused; those that only lie
between their rows are not.  On the CPU, with host tensors that say they are on a device and nothing launched."""

from __future__ import annotations

import random

import pytest
import torch

from fie_amd import beam
from fie_amd.beam import reorder_states


class OnDevice(torch.Tensor):
    def get_device(self):
        return 0


@pytest.fixture
def launches(monkeypatch):
    got = []
    monkeypatch.setattr(beam, "_reorder", lambda index, args: got.append(args))
    return got


def on_device(*shape):
    return torch.zeros(shape).as_subclass(OnDevice)


def test_buffers_in_each_others_place(launches):
    a, b, c = (on_device(4, 6) for _ in range(3))
    p = torch.zeros(4, dtype=torch.int32).as_subclass(OnDevice)
    room = on_device(4, 20)
    for states, out in (([a, b], [b, a]), ([a, b], [b, c]), ([a, b], [c, a]), ([a, b], [c, c]), ([a, b, c], [room[:, :6], c, room[:, 6:12]]),
                        ([a, b], [room[:, :6], room[:, 5:11]]), ([room[:, :6], a], [b, room[:, 3:9]]), ([a[:, :3], b], [c[:, :3], a]),
                        ([a], [a])):
        with pytest.raises(ValueError, match="overlap"):
            reorder_states(states, p, out=out)
    with pytest.raises(ValueError, match="overlap"):
        reorder_states([p.clone()], p, out=[p])
    assert not launches
    # the same state for two outputs, columns of one buffer, and outputs between the rows of states
    reorder_states([a, a], p, out=[b, c])
    reorder_states([a, b, c], p, out=[room[:, :6], room[:, 6:12], room[:, 14:]])
    reorder_states([room[:, :6], room[:, 2:8]], p, out=[room[:, 8:14], room[:, 14:]])
    reorder_states([a[:1].expand(4, 6), b], p, out=[c, room[:, 3:9]])
    tall = on_device(8, 10)
    reorder_states([tall[:4, :5], a], p, out=[tall[4:, :5], tall[4:, 5:10][:, :5].new_zeros(4, 6)])
    reorder_states([tall[:4, :5], tall[:4, 5:]], p, out=[tall[4:, :5], tall[4:, 5:]])
    assert len(launches) == 6


def test_columns_of_two_buffers(launches):
    p = torch.zeros(4, dtype=torch.int32).as_subclass(OnDevice)
    a, b = on_device(4, 120), on_device(4, 121)
    columns = lambda t, at=0: [t[:, at + 10 * i:at + 10 * i + 10] for i in range(12)]  # noqa: E731
    reorder_states(columns(a), p, out=columns(b))
    reorder_states(columns(b, 1), p, out=columns(a))
    reorder_states([a[:, :10]] * 11, p, out=columns(b)[:11])
    assert len(launches) == 3
    for out in (columns(b)[:11] + [b[:, 109:119]], columns(b)[:11] + [b[:, 0:10]], columns(a)[1:] + [b[:, :10]]):
        with pytest.raises(ValueError):
            reorder_states(columns(a), p, out=out)
    one = on_device(1, 40)                              # single rows: stretches of memory
    reorder_states([one[:, :2]] * 10, p[:1], out=[one[:, 2 + 3 * i:4 + 3 * i] for i in range(10)])
    with pytest.raises(ValueError):
        reorder_states([one[:, :2]] * 10, p[:1], out=[one[:, 1 + i:3 + i] for i in range(10)])


@pytest.mark.parametrize("most, size", [(3, 160), (12, 600)])
def test_any_views_of_one_buffer(launches, most, size):
    """Against the elements themselves, all rows at one stride."""
    rng = random.Random(most)
    seen = [0, 0]
    for _ in range(2000):
        room = torch.zeros(size).as_subclass(OnDevice)
        stride, n, kinds = rng.choice((8, 10, 12)) if most < 9 else rng.choice((60, 100)), rng.randint(1, 4), rng.randint(1, most)

        def view(width):
            rows = n
            return room.as_strided((rows, width), (stride, 1), rng.randrange(size - stride * (rows - 1) - width))

        widths = [rng.randint(1, 4) for _ in range(kinds)]
        states, outs = [view(w) for w in widths], [view(w) for w in widths]
        elements = lambda t: {t.storage_offset() + r * stride + c for r in range(n) for c in range(t.shape[1])}  # noqa: E731
        clash = any(elements(o) & elements(t) for i, o in enumerate(outs) for t in states + outs[:i])
        seen[clash] += 1
        parents = torch.zeros(n, dtype=torch.int32).as_subclass(OnDevice)
        if clash:
            with pytest.raises(ValueError):
                reorder_states(states, parents, out=outs)
        else:
            reorder_states(states, parents, out=outs)
    assert min(seen) > 200
