"""select_blocks for as many lists as a launch of one kernel takes, and its refusal
past that."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import target
from tests.test_gpu_kv4 import BF, data, ints, np64
from tests.test_gpu_kv4_blocks import bounds_of, filled

pytestmark = pytest.mark.gpu


def test_prompts_of_many_rows(gpu):
    """64 rows of 8,192 tokens and 8 KV heads, 2^22 lists, and twice as many rows; they
    share their pages."""
    n, heads, d, page, blocks = 8192, 8, 64, 256, 4
    c, table, kq, _, _ = filled(gpu, 1, [n], heads, d, page, BF, 1)
    q = data(gpu, 1, n, heads, d, BF, 2)
    one = c.select_blocks(q, table, ints([n], gpu), None, blocks)
    at = [0, 31, 32, 4099, n - 2, n - 1]
    bounds = bounds_of(kq, [n], page, table.shape[1])
    for i in at:
        exp = target.select_blocks(np64(q[:, i:i + 1]), bounds, [i + 1], [1], n,
                                   blocks, 1, 2)
        np.testing.assert_array_equal(one[:, i:i + 1].cpu().numpy(), exp)
    for b in (64, 128):
        got = c.select_blocks(q.expand(b, -1, -1, -1), table.expand(b, -1),
                              ints([n] * b, gpu), None, blocks)
        assert torch.equal(got, one.expand(b, -1, -1, -1))


def test_more_lists_than_a_launch_takes(gpu):
    """Said by name, with and without a workspace."""
    from suffixgpu_amd._lib import SuffixGPUError
    c, table, _, _, _ = filled(gpu, 1, [64], 1, 64, 64, BF, 3, cap=64 * 1024)
    q = torch.zeros(1, 1, 1, 64, dtype=BF, device=gpu)
    for b, t, tab in ((1024, 4096, table), (4096, 32768, table[:, :1])):
        tab = tab[:1].expand(b, -1)
        with pytest.raises(SuffixGPUError, match="lists"):
            c.select_blocks(q.expand(b, t, -1, -1), tab, ints([64] * b, gpu),
                            None, 3)
