"""select_blocks with more blocks of NaN than a query asks for: their keys lie far
above all others, at the end of the range that the choice searches."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import target
from tests.test_gpu_kv4 import BF, ints, np64
from tests.test_gpu_kv4_blocks import bounds_of, filled

pytestmark = pytest.mark.gpu

D, NANS = 64, 20


def keys(blocks, least, seed):
    """[1, 32 blocks, 1, D]: 20 blocks of NaN; with a query of ones the others
    score `least`, and from there on away from zero or past it."""
    g = torch.Generator().manual_seed(seed)
    top = torch.rand(blocks, generator=g) * 8 * abs(least)
    # (of 64 channels, the query packed to 64 of each)
    top = (least + top) / (64 * D)
    top[blocks // 2] = least / (64 * D)
    k = top[:, None, None].expand(blocks, 32, D).contiguous()
    for i in torch.randperm(blocks - 4, generator=g)[:NANS].tolist():
        k[2 + i, i % 32, i % D] = float("nan")
    return k.view(1, -1, 1, D).to(BF)


# choices by a wave over up to 256, 512 and 1,024 blocks; by a workgroup, in one
# launch and in two, in memory
@pytest.mark.parametrize("least", [-10.0, -5000.0, 0.5, 0.9, 16.0, 64.0])
@pytest.mark.parametrize("t,blocks,cap", [
    (1, 60, 256), (3, 250, 256), (3, 490, 512), (131, 1000, 1024),
    (131, 60, 1024), (1, 490, 512), (1, 1000, 1024), (1, 4000, 4096),
    (2, 4200, 5000), (1, 16500, 17000)])
def test_more_blocks_of_nan_than_wanted(gpu, least, t, blocks, cap):
    b = 2
    k = torch.cat([keys(blocks, least, 5), keys(blocks, least, 6)]).to(gpu)
    lens = [32 * blocks, 32 * blocks - 7]
    c, table, kq, _, _ = filled(gpu, b, lens, 1, D, 128, BF, 7, cap=32 * cap, k=k)
    q = torch.ones(b, t, 2, D, dtype=BF, device=gpu)
    bounds = bounds_of(kq, lens, 128, table.shape[1])
    for n, first, recent in ((11, 1, 2), (3, 0, 2), (30, 1, 2)):
        got = c.select_blocks(q, table, ints(lens, gpu), None, n, first, recent)
        # (tokens that see the same blocks choose the same)
        few = min(t, 2)
        exp = target.select_blocks(np64(q)[:, :few], bounds,
                                   [x - t + few for x in lens], [few] * b,
                                   table.shape[1] * 128, n, first, recent)
        got = got.cpu().numpy()
        np.testing.assert_array_equal(got[:, :few], exp)
        every = target.select_blocks(np64(q)[:, -1:], bounds, lens, [1] * b,
                                     table.shape[1] * 128, n, first, recent)
        np.testing.assert_array_equal(got[:, -1:], every)
        # every list ascends, with -1 behind: none holds another's entries
        flat = got.reshape(-1, n)
        full = flat[:, 1:] > flat[:, :-1]
        assert (full | (flat[:, 1:] == -1)).all()
