"""first_beams gives what beam_step takes, whatever torch's default type is."""

from __future__ import annotations

import pytest
import torch

from fie_amd.beam import first_beams


@pytest.mark.parametrize("default", [torch.float64, torch.float16, torch.bfloat16])
def test_types_do_not_hang_on_the_default(default):
    want = [t.dtype for t in first_beams(2, 3, "cpu")]
    torch.set_default_dtype(default)
    try:
        got = [t.dtype for t in first_beams(2, 3, "cpu")]
    finally:
        torch.set_default_dtype(torch.float32)
    assert got == want == [torch.float32, torch.int32, torch.bool, torch.float32, torch.int32]
