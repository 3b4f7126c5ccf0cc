"""select_blocks in the forms that its kernels have for rows of some length and lists
of some number, against the definition in whole numbers."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import target
from tests.test_gpu_kv4 import BF, HF, data, ints, np64
from tests.test_gpu_kv4_blocks import bounds_of, filled

pytestmark = pytest.mark.gpu


# up to 256, 512 and 1,024 blocks; by a wave, by a workgroup, in two launches
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("b,t,heads,d,cap,lens", [
    (3, 1, 2, 64, 12000, [12000, 9000, 33]),
    (2, 2, 1, 128, 16384, [16384, 16353]),
    (2, 5, 2, 64, 16384, [16000, 8200]),
    (2, 17, 8, 64, 20000, [20000, 150]),
    (2, 16, 8, 64, 20000, [20000, 150]),
    (1, 33, 8, 128, 32768, [32768]),
    (2, 3, 1, 256, 32768, [32768, 700])])
def test_forms(gpu, dtype, b, t, heads, d, cap, lens):
    c, table, kq, _, _ = filled(gpu, b, lens, heads, d, 256, dtype, 100 + t, cap,
                                holes=[(0, 7)])
    q = data(gpu, b, t, 2 * heads, d, dtype, 101)
    bounds = bounds_of(kq, lens, 256, table.shape[1], [(0, 7)])
    ql = [t] * (b - 1) + [max(1, t - 1)]
    for n, first, recent in ((40, 1, 2), (3, 0, 1)):
        got = c.select_blocks(q, table, ints(lens, gpu), ints(ql, gpu), n, first,
                              recent)
        exp = target.select_blocks(np64(q), bounds, lens, ql,
                                   table.shape[1] * 256, n, first, recent)
        np.testing.assert_array_equal(got.cpu().numpy(), exp)


@pytest.mark.parametrize("t", [1, 2])
def test_many_rows_of_one_token(gpu, t):
    """More than 256 lists of tables of up to 1,024 blocks, most rows short."""
    from suffixgpu_amd import KV4Cache
    b, d, page, n = 262, 64, 256, 30000
    width = -(-n // page)
    c = KV4Cache(2 * width + b, 1, d, page_size=page, device=gpu, bounds=True)
    c.pages.fill_(255)
    table = torch.full((b, width), -1, dtype=torch.int32)
    table[:2] = torch.randperm(2 * width).view(2, width)
    table[2:, 0] = torch.arange(2 * width, 2 * width + b - 2)
    table = table.to(gpu)
    long_, short = data(gpu, 2, n, 1, d, BF, 102), data(gpu, b - 2, 200, 1, d,
                                                       BF, 103)
    c.append(long_, long_, table[:2], ints([0, 0], gpu))
    c.append(short, short, table[2:], ints([0] * (b - 2), gpu))
    lens = [n, n - 7000] + [200] * (b - 2)
    q = data(gpu, b, t, 3, d, BF, 104)
    got = c.select_blocks(q, table, ints(lens, gpu), None, 50).cpu().numpy()
    for rows, k in ((slice(0, 2), long_), (slice(2, b), short)):
        exp = target.select_blocks(
            np64(q)[rows], bounds_of(target.quantize_k(np64(k), False),
                                     lens[rows], page, width),
            lens[rows], [t] * b, width * page, 50, 1, 2)
        np.testing.assert_array_equal(got[rows], exp)


@pytest.mark.parametrize("t,cap", [(1, 12000), (2, 32768), (5, 12000),
                                   (70, 32768)])
def test_ties(gpu, t, cap):
    """Equal keys, keys that differ in their last digits, no query at all: more
    than a wave's lanes hold are equal."""
    b, d, n = 4, 64, 9
    lens = [11900] * b
    k = torch.ones(b, 11900, 1, d, dtype=BF, device=gpu)
    k[2, 320] = float("nan")
    k[3, 400:464] = 2.0
    k[1, 2000:9000:3, 0, 1] = 1.5
    c, table, kq, _, _ = filled(gpu, b, lens, 1, d, 64, BF, 105, cap=cap, k=k)
    q = data(gpu, b, t, 2, d, BF, 106)
    q[0] = 0.0
    q[2, 0, 0, 7] = float("nan")
    got = c.select_blocks(q, table, ints(lens, gpu), None, n, 1, 2)
    exp = target.select_blocks(np64(q), bounds_of(kq, lens, 64, table.shape[1]),
                               lens, [t] * b, cap, n, 1, 2)
    np.testing.assert_array_equal(got.cpu().numpy(), exp)
    for blocks in (100, 371, 400):
        got = c.select_blocks(q, table, ints(lens, gpu), None, blocks, 1, 2)
        exp = target.select_blocks(np64(q)[:, :2],
                                   bounds_of(kq, lens, 64, table.shape[1]),
                                   [x - t + min(t, 2) for x in lens],
                                   [min(t, 2)] * b, cap, blocks, 1, 2)
        np.testing.assert_array_equal(got.cpu().numpy()[:, :2], exp)
