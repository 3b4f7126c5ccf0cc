"""Bounds of rows that are not written in order: of what an append's last block holds
behind its tokens, and whole again by update_bounds."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import target
from tests.test_gpu_kv4 import BF, HF, data, ints, np64
from tests.test_gpu_kv4_blocks import bounds_of, make

pytestmark = pytest.mark.gpu


def check(c, table, kq, ends):
    """ends[i][j]: how many tokens block j of row i counts."""
    lo, hi = (np64(x) for x in c.bounds(table))
    for i, row in enumerate(ends):
        for j, n in enumerate(row):
            for a in range(kq.shape[2]):
                k = kq[i, 32 * j:32 * j + n, a]
                x, y, u = target.key_bounds(k)
                np.testing.assert_array_equal(lo[i, j, a], x * 2.0 ** u)
                np.testing.assert_array_equal(hi[i, j, a], y * 2.0 ** u)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("first,then,ends,again", [
    # out of order: 48 .. 99, then 0 .. 47
    ((48, 52), (0, 48), [32, 16, 32, 4], 0),
    # written again inside a longer row: 10 .. 19 of 100
    ((0, 100), (10, 10), [20, 32, 32, 4], 10),
    # up to a block's end: whole
    ((0, 100), (30, 34), [32, 32, 32, 4], 30)])
def test_a_row_that_goes_on_behind_an_append(gpu, dtype, first, then, ends, again):
    b, heads, d, n, page = 2, 2, 64, 100, 32
    c, table = make(gpu, b, n, heads, d, page, dtype, 1)
    k = data(gpu, b, n, heads, d, dtype, 2)
    k[:, 50:] *= 3
    old = data(gpu, b, n, heads, d, dtype, 3) * 9
    for i, (at, m) in enumerate((first, then)):
        x = k[:, at:at + m]
        if i == 0 and then[0] > at:   # what is written again is other keys at first
            x = torch.cat([x[:, :then[0]], old[:, :then[1]],
                           x[:, then[0] + then[1]:]], 1)
        c.append(x, x, table, ints([at] * b, gpu))
    kq = target.quantize_k(np64(k), dtype == HF)
    check(c, table, kq, [ends] * b)
    c.update_bounds(table, ints([again] * b, gpu), n, ints([n - again] * b, gpu))
    check(c, table, kq, [[32, 32, 32, 4]] * b)
    # a query then finds what it would have found
    q = data(gpu, b, 1, heads * 2, d, dtype, 4)
    got = c.select_blocks(q, table, ints([n] * b, gpu), None, 2, 0, 1)
    exp = target.select_blocks(np64(q), bounds_of(kq, [n] * b, page,
                                                  table.shape[1]),
                               [n] * b, [1] * b, table.shape[1] * page, 2, 0, 1)
    np.testing.assert_array_equal(got.cpu().numpy(), exp)
