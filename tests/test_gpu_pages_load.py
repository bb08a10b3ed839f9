"""Pages given to a pool as 64-bit numbers, on an MI355X: what is no page or length of it is refused, not cut to 32 bits."""

from __future__ import annotations

import pytest
import torch

from fie_amd.pages import CachePages

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("where", ["cpu", DEV])
def test_numbers_past_32_bits(where):
    pool = CachePages(20, 4, 2, 5, DEV)
    table, lengths = torch.tensor([[3, 4, -1, -1, -1], [3, 7, -1, -1, -1]], device=where), torch.tensor([7, 6], device=where)
    pool.load(table, lengths)
    kept = pool.state.clone()
    for bad_table, bad_lengths in ((table + torch.tensor([1 << 32, 0, 0, 0, 0], device=where), lengths),
                                   (table - torch.tensor([0, 1 << 32, 0, 0, 0], device=where), lengths),
                                   (table, lengths + (1 << 32)), (table, lengths - (1 << 32))):
        with pytest.raises(ValueError):
            pool.load(bad_table, bad_lengths)
        assert torch.equal(pool.state, kept)
    # what is past a row's pages may be anything
    pool.load(table + torch.tensor([0, 0, 1 << 32, -(1 << 40), 9], device=where), lengths)
    assert torch.equal(pool.state, kept)


def test_lengths_past_31_bits_of_large_pages():
    """max_pages * page_size is 2^32, a length is an int32."""
    pool = CachePages(1 << 16, 1 << 16, 1, 1 << 16, DEV)
    table = torch.arange(1 << 16)[None]
    pool.load(table, torch.tensor([(1 << 31) - 1]))
    assert int(pool.lengths[0]) == (1 << 31) - 1 and pool.free_pages() == 1 << 15
    with pytest.raises(ValueError):
        pool.load(table, torch.tensor([1 << 31]))
    with pytest.raises(ValueError):
        pool.load(table, torch.tensor([float("nan")]))
    with pytest.raises(ValueError):
        pool.load(table, torch.tensor([2.0 ** 31]))     # fp32 holds no 2^31 - 1 to compare it with
