"""A step that is refused for its sizes has a workspace of 0 bytes.  On the CPU."""

from __future__ import annotations

import struct

import pytest

from fie_amd import _lib


def beam_args(**kw):
    a = dict(row_stride=1 << 31, workspace=256, workspace_bytes=1 << 40, length_penalty=1.0, requests=1, beams=4, vocab=100, dtype=0,
             early=0, min_tokens=0, pad=0, steps=0, eos_count=0)
    assert set(kw) <= set(a)
    return struct.pack(_lib.BEAM_ARGS, *[256] * 13, 0, 0, *{**a, **kw}.values(), *[0] * 16, 0)


@pytest.mark.parametrize("kw", [dict(vocab=(1 << 31) - 1), dict(vocab=524289), dict(requests=1 << 30), dict(requests=(1 << 31) - 1, beams=64),
                                dict(requests=16384), dict(eos_count=17), dict(eos_count=(1 << 31) - 1), dict(beams=65), dict(beams=-1)])
def test_no_workspace_for_what_is_refused(kw):
    lib = _lib.load()
    assert lib.fie_beam_workspace_size(beam_args()) > 0
    assert lib.fie_beam_workspace_size(beam_args(**kw)) == 0
