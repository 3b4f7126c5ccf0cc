"""attend_blocks where the blocks of a tile's tokens are joined over many tiles, and
over rows longer than one window."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import target
from tests.test_gpu_kv4 import BF, data, ints, np64
from tests.test_gpu_kv4_blocks import filled, make

pytestmark = pytest.mark.gpu


def check_rows(out, q, sel, kq, vq, vs, kv_len, t, rows):
    """As check_blocks, of some (batch row, token, query head)."""
    heads, hq = sel.shape[2], q.shape[2]
    g = hq // heads
    out, q, sel = np64(out), np64(q), sel.cpu().numpy()
    rel, tiny = target.ulp16(False)
    for i, j, a in rows:
        see = min(kv_len[i] - t + j + 1, kq.shape[1])
        at = [p for x in sorted(set(sel[i, j, a // g].tolist())) if x >= 0
              for p in range(32 * x, min(32 * x + 32, see))]
        if not at:
            assert (out[i, j, a] == 0).all()
            continue
        exp, bound = target._attend_row(q[i, j, a], kq[i, at, a // g],
                                        vq[i, at, a // g],
                                        vs[i, at, a // g, 0],
                                        q.shape[-1] ** -0.5)
        err = np.abs(out[i, j, a] - exp)
        assert (err <= bound + rel * (np.abs(exp) + bound) + tiny).all(), (
            i, j, a, err.max())


@pytest.mark.parametrize("heads,group,t", [(8, 4, 1100), (8, 3, 1300)])
def test_many_tiles(gpu, heads, group, t):
    """More than 2,048 tiles, the last of them of fewer tokens."""
    d, n, lens = 64, 9, [t + 500]
    c, table, kq, vq, vs = filled(gpu, 1, lens, heads, d, 64, BF, 90)
    q = data(gpu, 1, t, heads * group, d, BF, 91)
    kv = ints(lens, gpu)
    g = torch.Generator().manual_seed(92)
    lists = [c.select_blocks(q, table, kv, None, n),
             torch.randint(-3, 55, (1, t, heads, n), generator=g,
                           dtype=torch.int32).to(gpu)]
    r = np.random.default_rng(93)
    rows = [(0, int(r.integers(t)), int(r.integers(heads * group)))
            for _ in range(150)] + [(0, t - 1, 0), (0, t - 2, 5), (0, 0, 1)]
    for sel in lists:
        out = c.attend_blocks(q, sel, table, kv)
        check_rows(out, q, sel, kq, vq, vs, lens, t, rows)
        assert torch.equal(out, c.attend_blocks(q, sel, table, kv))


def test_rows_of_several_windows(gpu):
    """Lists over 16,000 blocks, in any order, each token its own."""
    b, d, n, t, group = 2, 64, 530000, 3, 5
    lens = [n, n - 200000]
    c, table = make(gpu, b, n, 1, d, 4096, BF, 94)
    g = torch.Generator(device=gpu).manual_seed(95)
    k = torch.randn(b, n, 1, d, generator=g, device=gpu).to(BF)
    c.append(k, k, table, ints([0, 0], gpu), ints(lens, gpu))
    kq = target.quantize_k(np64(k), False)
    vq, vs = target.quantize_v(np64(k))
    q = data(gpu, b, t, group, d, BF, 96)
    h = torch.Generator().manual_seed(97)
    sel = torch.randint(-100, 17000, (b, t, 1, 70), generator=h,
                        dtype=torch.int32)
    sel[:, :, :, 3] = 8191
    sel[:, :, :, 4] = 8192
    sel[:, 1:, :, :20] = sel[:, :1, :, :20]
    sel = sel.to(gpu)
    out = c.attend_blocks(q, sel, table, ints(lens, gpu))
    check_rows(out, q, sel, kq, vq, vs, lens, t,
               [(i, j, a) for i in range(b) for j in range(t)
                for a in range(group)])
