"""PagePool where its documentation has an exception: starts below zero, and lengths
put back when pages had run short."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import target

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_slots_of_rows_not_in_use(gpu, dtype):
    """A negative start names no position of its row, not even those that would
    follow it from 0 on."""
    from suffixgpu_amd import PagePool
    pool = PagePool(8, 4, 3, page_size=4, device=gpu)
    pool.resize(torch.tensor([12, 5, 9], dtype=dtype, device=gpu))
    o = target.Pages(8, 4, 3, 4)
    o.resize([12, 5, 9])
    for start in ([-1, 0, -3], [2, -1, -12], [-2 ** 31, 4, -1]):
        got = pool.slots(torch.tensor(start, dtype=dtype, device=gpu), 9)
        np.testing.assert_array_equal(got.cpu().numpy(), o.slots(start, 9))
        for r, s in enumerate(start):
            if s < 0:
                assert (got[r] == -1).all()


def test_lengths_put_back_after_pages_ran_short(gpu):
    """Row 0 asked for two pages and had one; what row 1 gives back goes to row 0
    when both ask again, whose lengths are as they were."""
    from suffixgpu_amd import PagePool

    def lens(*x):
        return torch.tensor(x, dtype=torch.int32, device=gpu)
    pool = PagePool(3, 2, 3, page_size=4, device=gpu)
    o = target.Pages(3, 2, 3, 4)
    for call in ((-1, 8), (8, 8), (8, 0), (8, 8)):
        room = pool.resize(lens(*call))
        assert room.tolist() == o.resize(list(call))
        np.testing.assert_array_equal(pool.table.cpu().numpy(), o.table())
    assert pool.held.tolist() == [2, 1]
    # where all had what they asked for, the pages come back (row 0's second page is
    # free from the next call on: row 1 has it then)
    pool.resize(lens(4, 8))
    assert pool.held.tolist() == [1, 1]
    pool.resize(lens(4, 8))
    assert pool.held.tolist() == [1, 2]
    before = pool.table.clone()
    pool.resize(lens(0, 12))
    pool.resize(lens(4, 8))
    assert torch.equal(pool.table, before)
