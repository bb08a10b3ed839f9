"""adapter_linear's out is base itself or has none of its memory.  On the CPU, with host tensors that say
they are on a device and nothing launched."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from fie_amd import adapters
from fie_amd.adapters import adapter_linear


class OnDevice(torch.Tensor):
    def get_device(self):
        return 0


def on_device(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype).as_subclass(OnDevice)


@pytest.fixture
def launches(monkeypatch):
    got = []
    monkeypatch.setattr(adapters, "_run", lambda index, args: got.append(args))
    monkeypatch.setattr(adapters, "_size", lambda args: 64)
    return got


def setup(dtype, tokens, k=4, n=6):
    some = on_device(1)
    bank = SimpleNamespace(k=k, n=n, index=0, adapters=2, dtype=dtype, a=some, b=some, scale=some, ranks=some, rank_pad=16, k_pad=64,
                           b_pitch=16, on_stream=lambda: None)
    return bank, SimpleNamespace(tokens=tokens, adapters=2, index=0, data=some, on_stream=lambda: None), on_device(tokens, k, dtype=dtype)


def test_base_in_outs_memory(launches):
    bank, plan, x = setup(torch.float32, 5)
    tall, wide = on_device(9, 6), on_device(5, 20)
    for base, out in ((tall[1:6], tall[:5]), (tall[:5], tall[4:]), (wide[:, :6], wide[:, 5:11]), (wide[:, 8:14], wide[:, 3:9]),
                      (tall[0].expand(5, 6), tall[:5]), (tall[2].expand(5, 6), tall[:5]), (tall[:5], tall.view(-1)[:54].view(3, 18)[:, :6][:1].expand(5, 6))):
        with pytest.raises(ValueError):
            adapter_linear(x, bank, plan, base=base, out=out)
    assert not launches
    for base, out in ((tall[:5], tall[:5]), (wide[:, :6], wide[:, 6:12]), (wide[:, 14:], wide[:, :6]), (tall[5].expand(5, 6), tall[:5]),
                      (on_device(5, 6), tall[:5])):
        assert adapter_linear(x, bank, plan, base=base, out=out) is out
    assert len(launches) == 5
    # one token: a row
    bank, plan, x = setup(torch.float32, 1)
    adapter_linear(x, bank, plan, base=wide[:1, :6], out=wide[:1, 6:12])
    with pytest.raises(ValueError):
        adapter_linear(x, bank, plan, base=wide[:1, :6], out=wide[:1, 5:11])


def test_base_of_another_type(launches):
    bank, plan, x = setup(torch.bfloat16, 5)
    room = on_device(5, 16)
    half = room.view(torch.bfloat16)
    with pytest.raises(ValueError):
        adapter_linear(x, bank, plan, base=room[:, :6], out=half[:, 10:16])
    adapter_linear(x, bank, plan, base=room[:, :6], out=half[:, 12:18])
    assert len(launches) == 1
