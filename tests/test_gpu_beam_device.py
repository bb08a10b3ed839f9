"""A search keeps the device that it was made on, named without a number, on an MI355X."""

from __future__ import annotations

import pytest
import torch

from fie_amd.beam import BeamSearch

pytestmark = pytest.mark.gpu


def test_the_device_has_a_number():
    search = BeamSearch("cuda", 2, 3, max_tokens=4)
    assert search.device == search.beams.scores.device == torch.device("cuda", torch.cuda.current_device())
    search.stop([1])
    search.restart([0, 1])
    assert search.beams.done.tolist() == [False, False]
