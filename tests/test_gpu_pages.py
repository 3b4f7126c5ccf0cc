"""PagePool against lists of pages (oracle/target.py)."""

from __future__ import annotations

import random

import numpy as np
import pytest
import torch

from oracle import target

pytestmark = pytest.mark.gpu


def ints(x, gpu, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=gpu)


def same(pool, o, n=None):
    np.testing.assert_array_equal(pool.table.cpu().numpy(), o.table())
    assert pool.held.tolist() == [len(r) for r in o.rows]
    assert pool.num_free.tolist() == [len(o.free)]
    assert pool._stack[:len(o.free)].tolist() == o.free


# one workgroup's tables, and larger ones
@pytest.mark.parametrize("rows,width,page,pages", [
    (1, 1, 1, 1), (5, 7, 16, 20), (64, 128, 64, 4000), (1500, 40, 32, 30000),
    (300, 900, 1, 200000), (4096, 64, 64, 100000), (3, 5, 65536, 0)])
def test_lengths_come_and_go(gpu, rows, width, page, pages):
    from suffixgpu_amd import PagePool
    pool = PagePool(pages, rows, width, page_size=page, device=gpu)
    o = target.Pages(pages, rows, width, page)
    r = random.Random(rows * 7 + width)
    same(pool, o)
    for step in range(8):
        n = rows if step % 3 else r.randint(1, rows)
        lens = []
        for i in range(n):
            kind = r.random()
            now = len(o.rows[i]) * page
            if kind < 0.2:
                lens.append(-r.randint(1, 9))
            elif kind < 0.3:
                lens.append(0)
            elif kind < 0.7:
                lens.append(max(0, now + r.randint(-2 * page, 3 * page)))
            else:
                lens.append(r.randint(0, page * (width + 2)))
        room = pool.resize(ints(lens, gpu, torch.int64 if step % 2
                                else torch.int32))
        assert room.dtype == torch.int32 and room.tolist() == o.resize(lens)
        same(pool, o)
        tokens = r.randint(1, 3 * page if page < 1000 else 50)
        start = [max(0, x - r.randint(0, tokens)) for x in lens]
        count = [r.randint(-1, tokens + 2) for _ in lens]
        np.testing.assert_array_equal(
            pool.slots(ints(start, gpu), tokens, ints(count, gpu)).cpu(),
            o.slots(start, tokens, count))
        np.testing.assert_array_equal(
            pool.slots(ints(start, gpu, torch.int64), tokens).cpu(),
            o.slots(start, tokens))


@pytest.mark.parametrize("rows,width", [(40, 30), (400, 700)])
def test_lengths_put_back_put_the_pages_back(gpu, rows, width):
    from suffixgpu_amd import PagePool
    page = 32
    pool = PagePool(rows * width // 2, rows, width, page_size=page, device=gpu)
    g = torch.Generator().manual_seed(1)

    def lens():
        return torch.randint(0, width * page, (rows,), generator=g,
                             dtype=torch.int32).to(gpu) // 3
    pool.resize(lens())
    a = lens()
    pool.resize(a)
    room = pool.resize(a)
    assert (room >= a).all()
    before = [t.clone() for t in (pool.table, pool.held, pool.num_free)]
    free = pool._stack[:int(pool.num_free)].clone()
    for b in (a + 17, lens() * 3, torch.zeros_like(a), lens()):
        pool.resize(b)
        pool.resize(a)
        for x, y in zip(before, (pool.table, pool.held, pool.num_free)):
            assert torch.equal(x, y)
        assert torch.equal(free, pool._stack[:len(free)])


def test_no_page_is_lost_or_twice(gpu):
    """Shortage, then everything back."""
    from suffixgpu_amd import PagePool
    pool = PagePool(1000, 64, 64, page_size=64, device=gpu)
    g = torch.Generator().manual_seed(2)
    for _ in range(30):
        lens = torch.randint(-1, 64 * 64, (64,), generator=g)
        room = pool.resize(lens.to(gpu))
        held = pool.table[pool.table >= 0]
        free = pool._stack[:int(pool.num_free)]
        both = torch.cat([held, free]).sort().values
        assert torch.equal(both, torch.arange(1000, device=gpu,
                                              dtype=torch.int32))
        assert torch.equal(room, pool.held * 64)
    assert pool.resize(torch.zeros(64, dtype=torch.int64,
                                   device=gpu)).sum() == 0
    assert int(pool.num_free) == 1000


def test_long_lengths_do_not_wrap(gpu):
    from suffixgpu_amd import PagePool
    pool = PagePool(50, 4, 20, page_size=64, device=gpu)
    big = 2 ** 63 - 1
    room = pool.resize(ints([big, -big, 5, big], gpu, torch.int64))
    assert room.tolist() == [20 * 64, 0, 64, 20 * 64]
    got = pool.slots(ints([big, 2 ** 62, -5, 63], gpu, torch.int64), 4)
    assert (got[:3] == -1).all()
    t = pool.table[3].tolist()
    assert got[3].tolist() == [t[0] * 64 + 63, t[1] * 64, t[1] * 64 + 1,
                               t[1] * 64 + 2]


def test_graph_replays(gpu):
    """A step's growth and trim, recorded once."""
    from suffixgpu_amd import PagePool
    rows, width, page = 100, 900, 32
    pool = PagePool(60000, rows, width, page_size=page, device=gpu)
    o = target.Pages(60000, rows, width, page)
    grow, trim = (torch.zeros(rows, dtype=torch.int32, device=gpu)
                  for _ in range(2))
    pool.resize(grow)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        room = pool.resize(grow)
        slots = pool.slots(trim, 9)
        pool.resize(trim)
    r = random.Random(3)
    lens = [0] * rows
    for _ in range(6):
        more = [x + r.randint(0, 300) for x in lens]
        kept = [r.randint(a, b) for a, b in zip(lens, more)]
        grow.copy_(ints(more, gpu))
        trim.copy_(ints(kept, gpu))
        g.replay()
        assert room.tolist() == o.resize(more)
        np.testing.assert_array_equal(slots.cpu(), o.slots(kept, 9))
        o.resize(kept)
        same(pool, o)
        lens = kept


def test_on_another_device(gpu, elsewhere):
    from suffixgpu_amd import PagePool
    pool = PagePool(10, 2, 4, device=torch.device("cuda", gpu.index))
    pool.resize(ints([65, 1], gpu))
    pool.slots(ints([0, 0], gpu), 1)
    assert elsewhere.count(gpu.index) >= 2
    assert pool.table[:, :2].tolist() == [[0, 1], [2, -1]]


def test_refusals(gpu):
    from suffixgpu_amd import PagePool
    from suffixgpu_amd._lib import SuffixGPUError
    for bad in (dict(page_size=48), dict(page_size=1 << 17), dict(rows=0),
                dict(rows=4097), dict(width=0), dict(width=1 << 25),
                dict(num_pages=-1)):
        kw = dict(num_pages=4, rows=2, width=2, page_size=64, device=gpu)
        kw.update(bad)
        with pytest.raises(ValueError):
            PagePool(**kw)
    pool = PagePool(4, 2, 2, device=gpu)
    one = ints([1, 2, 3], gpu)
    for bad in (lambda: pool.resize(one), lambda: pool.resize(one[:2].float()),
                lambda: pool.resize(one[:2, None]),
                lambda: pool.resize(one[:2] > 0),
                lambda: pool.slots(one[:2], 3, one[:1]),
                lambda: pool.slots(one, 3)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(SuffixGPUError):
        pool.resize(one[:2].cpu())
    assert pool.resize(one[:0]).shape == (0,)
    assert pool.slots(one[:2], 0).shape == (2, 0)
