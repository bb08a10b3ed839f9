"""What is more than one launch holds is refused before it.  On the CPU: no call here reaches a launch."""

from __future__ import annotations

import struct

import pytest

from fie_amd import _lib


def refused(name, args, text):
    lib = _lib.load()
    assert getattr(lib, name)(args, None) == _lib.FIE_E_ARG
    assert text in lib.fie_sampler_last_error(), lib.fie_sampler_last_error()


def test_states_of_2_to_24_pieces():
    """256 threads each: 2^32, one more than a launch's count of threads can say."""
    row = 1 << 38                       # 2^24 pieces of 16 KB, but for the 15 bytes in front
    for bytes_ in (row - 15, row):
        refused("fie_reorder_states", struct.pack(_lib.STATES_ARGS + _lib.STATE_ARGS, 256, 1, 1, 256, 256, bytes_, bytes_, bytes_, 1), b"one launch")


@pytest.mark.parametrize("count, outer, token", [(1 << 12, 1 << 12, 16),        # 2^24 pieces
                                                 (1 << 16, 1 << 16, 16),        # 2^32: none in 32 bits
                                                 (3 << 15, 3 << 15, 16),        # 9 * 2^30, 2^30 in 32 bits
                                                 ((1 << 31) - 1, (1 << 31) - 1, 1 << 30)])
def test_pages_of_too_many_pieces(count, outer, token):
    args = struct.pack(_lib.PAGES_ARGS + _lib.GROUP_ARGS * 8, 256, 256, 1 << 20, 20, 65536 if token > 16 else 4, 3, 6, *[256] * 6, 2, 1,
                       256, 64, 64, token, count, outer, 0, 0, *[0] * 56)
    for name in ("fie_pages_step", "fie_pages_compact", "fie_pages_copy"):
        refused(name, args, b"too large")
