"""Caches whose pages lie between each other, on an MI355X: [heads, pages, page_size, dim] seen as [pages, heads, page_size, dim]."""

from __future__ import annotations

import pytest
import torch

from fie_amd.pages import CachePages

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("dim", [8, 7])
def test_heads_in_front_of_pages(dim):
    pages, page, heads = 12, 4, 3
    room = torch.randn(heads, pages, page, dim, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).half()
    want = room.clone()
    pool = CachePages(pages, page, 2, 4, DEV, caches=[room.transpose(0, 1)], token_dim=2)
    assert pool.step(i32([6, 0])).all() and pool.step(i32([6, 6]), i32([0, 0])).all() and pool.step(i32([7, 7])).all()
    assert pool.table[:, :2].tolist() == [[0, 1], [0, 2]]
    want[:, 2, :2] = want[:, 1, :2]
    assert torch.equal(room, want)
    pool.copy_pages(i32([0, 5]), i32([11, 3]))
    want[:, 11], want[:, 3] = want[:, 0], want[:, 5]
    assert torch.equal(room, want)


def test_pages_that_do_overlap_are_refused():
    pool = CachePages(12, 4, 2, 4, DEV)
    flat = torch.zeros(4096, device=DEV)
    for stride in ((31, 1000, 8, 1), (32, 32 * 12 - 1, 8, 1), (63, 32, 8, 1), (0, 32, 8, 1)):
        with pytest.raises(ValueError):
            pool.add_caches([flat.as_strided((12, 2, 4, 8), stride)], 2)
    pool.add_caches([flat.as_strided((12, 2, 4, 8), (32, 32 * 12, 8, 1)), flat.as_strided((12, 2, 4, 8), (64, 32, 8, 1))], 2)
