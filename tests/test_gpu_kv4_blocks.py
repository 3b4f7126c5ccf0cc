"""KV4Cache's bounds, select_blocks and attend_blocks against the definitions in
64 bits and whole numbers (oracle/target.py)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import target
from tests.test_gpu_kv4 import BF, HF, check_attend, data, ints, np64

pytestmark = pytest.mark.gpu


def make(gpu, b, positions, heads, d, page, dtype, seed, holes=()):
    """A cache with bounds, all bytes garbage, and a shuffled table; holes: (row,
    page) without a page."""
    from suffixgpu_amd import KV4Cache
    width = -(-positions // page)
    c = KV4Cache(b * width, heads, d, page_size=page, dtype=dtype, device=gpu,
                 bounds=True)
    c.pages.fill_(255)
    c._range.fill_(77)
    c._unit.fill_(3)
    g = torch.Generator().manual_seed(seed)
    table = torch.randperm(b * width, generator=g).to(torch.int32)
    table = table.view(b, width)
    for r, p in holes:
        table[r, p] = -1 if (r + p) % 2 else b * width
    return c, table.to(gpu)


def filled(gpu, b, lens, heads, d, page, dtype, seed, cap=None, holes=(),
           k=None):
    n = max(max(lens), 1)
    c, table = make(gpu, b, cap or n, heads, d, page, dtype, seed, holes)
    if k is None:
        k = data(gpu, b, n, heads, d, dtype, seed + 1)
    v = data(gpu, b, n, heads, d, dtype, seed + 2)
    c.append(k, v, table, ints([0] * b, gpu), ints(lens, gpu))
    kq = target.quantize_k(np64(k), dtype == HF)
    vq, vs = target.quantize_v(np64(v))
    return c, table, kq, vq, vs


def bounds_of(kq, lens, page, width, holes=()):
    """bounds[i][j][a] as target.select_blocks takes them; garbage blocks (from a
    row's end on) are never asked for."""
    out = []
    for i, n in enumerate(lens):
        row = []
        for j in range(width * page // 32):
            if (i, j * 32 // page) in holes:
                row.append([None] * kq.shape[2])
            elif j * 32 < n:
                row.append([target.key_bounds(kq[i, 32 * j:min(32 * j + 32, n),
                                                 a])
                            for a in range(kq.shape[2])])
            else:
                row.append([(0, 0, 0)] * kq.shape[2])
        out.append(row)
    return out


# ------------------------------------------------------------------ bounds
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page,lens", [(32, [1, 32, 70]), (64, [33, 100, 0]),
                                       (256, [300, 31, 257])])
def test_bounds_are_the_stored_keys(gpu, dtype, d, page, lens):
    b, heads = 3, 2
    c, table, kq, _, _ = filled(gpu, b, lens, heads, d, page, dtype, 3, cap=320)
    lo, hi = (np64(x) for x in c.bounds(table))
    for i in range(b):
        for j in range(-(-lens[i] // 32)):
            for a in range(heads):
                k = kq[i, 32 * j:min(32 * j + 32, lens[i]), a]
                x, y, u = target.key_bounds(k)
                np.testing.assert_array_equal(lo[i, j, a], x * 2.0 ** u)
                np.testing.assert_array_equal(hi[i, j, a], y * 2.0 ** u)
                assert (lo[i, j, a] <= k.min(axis=0)).all()
                assert (hi[i, j, a] >= k.max(axis=0)).all()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_bounds_of_extreme_keys(gpu, dtype):
    d = 64
    tops = (65504.0, 1e-7, 6e-5, 0.0, 1.0) if dtype == HF else (
        3e38, 1e-38, 1e-30, 0.0, 2.0 ** 100, 2.0 ** 107, 2.0 ** -94, 1e-40)
    g = torch.Generator().manual_seed(1)
    k = torch.rand(1, 32 * len(tops), 1, d, generator=g) * 2 - 1
    for i, t in enumerate(tops):
        k[:, 32 * i:32 * i + 32] *= t
        k[:, 32 * i + 5, :, 40:] *= 2.0 ** -9
    k = k.to(dtype).to(gpu)
    c, table, kq, _, _ = filled(gpu, 1, [k.shape[1]], 1, d, 32, dtype, 4, k=k)
    unit = c._unit[table[0].long()].view(-1).tolist()
    rng = c._range[table[0].long()].view(-1, 2 * d).cpu().numpy()
    for j in range(len(tops)):
        lo, hi, u = target.key_bounds(kq[0, 32 * j:32 * j + 32, 0])
        assert unit[j] == u, (j, unit[j], u)
        np.testing.assert_array_equal(rng[j, :d], lo)
        np.testing.assert_array_equal(rng[j, d:], hi)


def test_bounds_follow_an_append_that_overwrites(gpu):
    """Rejected drafts, large ones, leave no trace once written over."""
    d, b = 128, 2
    c, table = make(gpu, b, 256, 2, d, 64, BF, 5)
    k = data(gpu, b, 200, 2, d, BF, 6)
    c.append(k, k, table, ints([0, 0], gpu), ints([100, 60], gpu))
    wild = k[:, :40] * 50
    c.append(wild, wild, table, ints([100, 60], gpu), ints([40, 33], gpu))
    c.append(k[:, 100:], k[:, 100:], table, ints([100, 60], gpu),
             ints([60, 68], gpu))
    stored, _ = c.read(table, ints([0, 0], gpu), 160)
    lo, hi = (np64(x) for x in c.bounds(table))
    for i, n in enumerate((160, 128)):
        for j in range(n // 32):
            x, y, u = target.key_bounds(np64(stored)[i, 32 * j:32 * j + 32, 1])
            np.testing.assert_array_equal(lo[i, j, 1], x * 2.0 ** u)
            np.testing.assert_array_equal(hi[i, j, 1], y * 2.0 ** u)


def test_bounds_of_nan_and_of_no_page(gpu):
    d = 64
    k = data(gpu, 1, 128, 1, d, BF, 7)
    k[0, 40, 0, 3] = float("nan")
    k[0, 70, 0, 50] = float("inf")
    c, table, _, _, _ = filled(gpu, 1, [128], 1, d, 32, BF, 8, k=k,
                               holes=[(0, 3)])
    lo, hi = c.bounds(table)
    assert torch.isnan(lo[0, 1]).all() and torch.isnan(hi[0, 2]).all()
    assert not torch.isnan(lo[0, 0]).any()
    assert (lo[0, 3] == 0).all() and (hi[0, 3] == 0).all()


def test_update_bounds_of_a_filled_pool(gpu):
    from suffixgpu_amd import KV4Cache
    c, table, kq, _, _ = filled(gpu, 2, [150, 90], 2, 128, 64, BF, 9, cap=192)
    e = KV4Cache(c.num_pages, 2, 128, device=gpu, pages=c.pages, bounds=True)
    e.update_bounds(table, ints([0, 0], gpu), 1 << 20, ints([150, 90], gpu))
    for x, y in zip(c.bounds(table), e.bounds(table)):
        assert torch.equal(x[0, :5], y[0, :5]) and torch.equal(x[1, :3],
                                                               y[1, :3])


# --------------------------------------------------------------- selection
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d,heads,group,t,page,lens,n,first,recent", [
    (128, 2, 4, 1, 64, [700, 33, 1], 5, 1, 2),
    (128, 1, 1, 17, 32, [900, 17, 300], 7, 0, 1),
    (64, 2, 3, 5, 128, [641, 640, 639], 4, 2, 2),
    (256, 1, 8, 3, 64, [512, 400, 64], 16, 1, 4),
    (128, 3, 2, 40, 256, [777, 40, 1000], 12, 3, 3),
    (64, 1, 20, 2, 32, [350, 2, 95], 1, 0, 1)])
def test_selection_is_the_definitions(gpu, dtype, d, heads, group, t, page,
                                      lens, n, first, recent):
    b = 3
    cap = 1024
    holes = [(0, 1), (2, 0)]
    c, table, kq, _, _ = filled(gpu, b, lens, heads, d, page, dtype, d + t, cap,
                                holes)
    q = data(gpu, b, t, heads * group, d, dtype, 11)
    q_len = [t, max(1, t - 1), t]
    got = c.select_blocks(q, table, ints(lens, gpu), ints(q_len, gpu), n, first,
                          recent)
    exp = target.select_blocks(
        np64(q), bounds_of(kq, lens, page, table.shape[1], holes), lens, q_len,
        table.shape[1] * page, n, first, recent)
    np.testing.assert_array_equal(got.cpu().numpy(), exp)


def test_selection_over_a_wide_table(gpu):
    """More blocks than a wave keeps, lists from none to all of them."""
    b, t, d = 4, 2, 64
    lens = [40000, 5, 33000, 1100]
    c, table, kq, _, _ = filled(gpu, b, lens, 1, d, 256, BF, 13, cap=40000,
                                holes=[(0, 3), (2, 100)])
    q = data(gpu, b, t, 2, d, BF, 14)
    bounds = bounds_of(kq, lens, 256, table.shape[1], [(0, 3), (2, 100)])
    for n, first, recent in ((64, 1, 2), (1030, 4, 1), (1300, 0, 5)):
        got = c.select_blocks(q, table, ints(lens, gpu), None, n, first, recent)
        exp = target.select_blocks(np64(q), bounds, lens, [t] * b,
                                   table.shape[1] * 256, n, first, recent)
        np.testing.assert_array_equal(got.cpu().numpy(), exp)


@pytest.mark.parametrize("n", [140000, 530000])
def test_selection_over_a_long_row(gpu, n):
    """Rows whose keys a workgroup keeps in many registers, or not at all."""
    b, d, page = 2, 64, 4096
    lens = [n, n - 40000]
    c, table = make(gpu, b, n, 1, d, page, BF, 45)
    g = torch.Generator(device=gpu).manual_seed(46)
    k = torch.randn(b, n, 1, d, generator=g, device=gpu).to(BF)
    k[:, 5000:6000] *= 4
    k[0, 9:70000:31] = 1.0
    c.append(k, k, table, ints([0, 0], gpu), ints(lens, gpu))
    kq = target.quantize_k(np64(k), False)
    q = data(gpu, b, 1, 2, d, BF, 47)
    kv = ints(lens, gpu)
    bounds = bounds_of(kq, lens, page, table.shape[1])
    for blocks, first, recent in ((70, 1, 2), (3000, 0, 1), (32768, 1, 1)):
        got = c.select_blocks(q, table, kv, None, blocks, first, recent)
        exp = target.select_blocks(np64(q), bounds, lens, [1] * b,
                                   table.shape[1] * page, blocks, first, recent)
        np.testing.assert_array_equal(got.cpu().numpy(), exp)


@pytest.mark.parametrize("cap", [1024, 40000, 140000, 530000])
def test_ties_go_to_the_lowest_blocks(gpu, cap):
    """Equal keys, zero queries, blocks of NaN, queries of NaN."""
    b, d, n = 4, 64, 9
    lens = [960] * b
    k = torch.ones(b, 960, 1, d, dtype=BF, device=gpu)
    k[2, 320] = float("nan")
    k[2, 640, 0, 5] = float("inf")
    k[3, 400:464] = 2.0
    c, table, kq, _, _ = filled(gpu, b, lens, 1, d, 64, BF, 15, cap=cap, k=k)
    q = data(gpu, b, 1, 2, d, BF, 16)
    q[1] = 0.0
    q[2, 0, 0, 7] = float("nan")
    q[3, 0, 1, 9] = -float("inf")
    got = c.select_blocks(q, table, ints(lens, gpu), None, n, 1, 2)
    exp = target.select_blocks(np64(q), bounds_of(kq, lens, 64, table.shape[1]),
                               lens, [1] * b, cap, n, 1, 2)
    np.testing.assert_array_equal(got.cpu().numpy(), exp)
    assert got[1, 0, 0].tolist() == [0, 1, 2, 3, 4, 5, 6, 28, 29]


def test_selection_past_the_table_and_before_it(gpu):
    """kv_len past the table, q_len past T, rows shorter than their q_len."""
    b, t, d = 4, 3, 64
    lens = [256, 256, 100, 0]
    c, table, kq, _, _ = filled(gpu, b, lens, 2, d, 32, BF, 17, cap=256)
    q = data(gpu, b, t, 2, d, BF, 18)
    kv, ql = [300, 258, 100, 1], [4, 3, 103, 3]
    got = c.select_blocks(q, table, ints(kv, gpu), ints(ql, gpu), 3, 0, 1)
    exp = target.select_blocks(np64(q), bounds_of(kq, [256] * 4, 32, 8), kv, ql,
                               256, 3, 0, 1)
    np.testing.assert_array_equal(got.cpu().numpy()[:3], exp[:3])
    assert (got[3, :2] == -1).all() and got[3, 2, 0].tolist() == [0, -1, -1]


def test_extreme_queries(gpu):
    b, d = 6, 128
    lens = [800] * b
    c, table, kq, _, _ = filled(gpu, b, lens, 1, d, 64, BF, 19)
    q = data(gpu, b, 1, 5, d, BF, 20)
    for i, s in enumerate((1e30, 1e-30, 2.0 ** -130, 1.0, 2.0 ** -7, 3e38 / 40)):
        q[i] *= s
    q[3, 0, 1:] = 0
    q[4, 0, :, 1:] = 0
    got = c.select_blocks(q, table, ints(lens, gpu), None, 6, 1, 1)
    exp = target.select_blocks(np64(q), bounds_of(kq, lens, 64, table.shape[1]),
                               lens, [1] * b, table.shape[1] * 64, 6, 1, 1)
    np.testing.assert_array_equal(got.cpu().numpy(), exp)


# --------------------------------------------------------------- attention
def check_blocks(out, q, sel, kq, vq, vs, kv_len, q_len, dtype, scale=None):
    exp, bound = target.attend_blocks(np64(q), sel.cpu().numpy(), kq, vq, vs,
                                      kv_len, q_len, scale)
    rel, tiny = target.ulp16(dtype == HF)
    err = np.abs(np64(out) - exp)
    tol = bound + rel * (np.abs(exp) + bound) + tiny
    tol = np.where(bound == 0, 0.0, tol)     # rows that see nothing are zeros
    bad = ~(err <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], err[bad][:5], tol[bad][:5])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d,heads,group,t,page,lens,n", [
    (128, 2, 4, 1, 64, [700, 33, 1], 5),
    (128, 1, 1, 17, 32, [600, 17, 300], 7),
    (64, 2, 3, 5, 128, [641, 640, 639], 40),
    (256, 1, 8, 3, 64, [512, 400, 64], 16),
    (64, 1, 20, 2, 32, [350, 2, 95], 3),
    (128, 1, 40, 1, 32, [300, 5, 64], 70)])
def test_attention_over_selected_blocks(gpu, dtype, d, heads, group, t, page,
                                        lens, n):
    b = 3
    c, table, kq, vq, vs = filled(gpu, b, lens, heads, d, page, dtype, d + n,
                                  cap=1024)
    q = data(gpu, b, t, heads * group, d, dtype, 21)
    q_len = [t, max(1, t - 1), t]
    kv, ql = ints(lens, gpu), ints(q_len, gpu)
    sel = c.select_blocks(q, table, kv, ql, n, 0, 1)
    out = c.attend_blocks(q, sel, table, kv, ql)
    check_blocks(out, q, sel, kq, vq, vs, lens, q_len, dtype)


def test_all_blocks_are_attend(gpu):
    b, t = 3, 5
    lens = [500, 77, 31]
    c, table, kq, vq, vs = filled(gpu, b, lens, 2, 128, 64, BF, 22)
    q = data(gpu, b, t, 8, 128, BF, 23)
    kv = ints(lens, gpu)
    sel = c.select_blocks(q, table, kv, None, 20)
    out = c.attend_blocks(q, sel, table, kv, None, 0.2)
    check_attend(out, q, kq, vq, vs, lens, [t] * b, BF, 0.2)


def test_lists_of_any_order(gpu):
    """Out of order, named twice, outside the table, past the query, without a
    page, none at all."""
    b, t, d, n = 2, 2, 64, 80
    lens = [400, 300]
    c, table, kq, vq, vs = filled(gpu, b, lens, 1, d, 32, HF, 24)
    q = data(gpu, b, t, 2, d, HF, 25)
    g = torch.Generator().manual_seed(26)
    sel = torch.randint(-20, 40, (b, t, 1, n), generator=g, dtype=torch.int32)
    sel[0, 1] = -1
    sel[1, 1, 0, :4] = torch.tensor([2 ** 31 - 1, -2 ** 31, 1 << 26, 13])
    sel = sel.to(gpu)
    out = c.attend_blocks(q, sel, table, ints(lens, gpu))
    check_blocks(out, q, sel, kq, vq, vs, lens, [t] * b, HF)
    # blocks without a page are none
    table[0, 3] = -1
    table[1, 2] = c.num_pages
    out = c.attend_blocks(q, sel, table, ints(lens, gpu))
    gone = sel.clone()
    gone[0][gone[0] == 3] = -1
    gone[1][gone[1] == 2] = -1
    check_blocks(out, q, gone, kq, vq, vs, lens, [t] * b, HF)


def test_many_lists_and_few_split_the_same(gpu):
    """One row alone, whose list is split, and the same row among many."""
    b, d, n = 300, 128, 64
    lens = [2100] * b
    c, table, kq, vq, vs = filled(gpu, 1, [2100], 4, d, 64, BF, 27)
    q = data(gpu, 1, 1, 16, d, BF, 28)
    kv = ints([2100], gpu)
    sel = c.select_blocks(q, table, kv, None, n)
    one = c.attend_blocks(q, sel, table, kv)
    check_blocks(one, q, sel, kq, vq, vs, [2100], [1], BF)
    many = c.attend_blocks(q.expand(b, -1, -1, -1),
                           sel.expand(b, -1, -1, -1).contiguous(),
                           table.expand(b, -1).contiguous(), ints(lens, gpu))
    assert (many == many[:1]).all()
    check_blocks(many[:1], q, sel, kq, vq, vs, [2100], [1], BF)


def test_values_of_zero_count(gpu):
    """Tokens of zero values beside large ones, as in attend: the sum of weights
    is taken again."""
    d = 64
    c, table = make(gpu, 1, 256, 1, d, 64, BF, 29)
    k = data(gpu, 1, 256, 1, d, BF, 30)
    v = torch.zeros(1, 256, 1, d, dtype=BF, device=gpu)
    v[0, 5] = 3e4
    c.append(k, v, table, ints([0], gpu))
    q = data(gpu, 1, 1, 4, d, BF, 31) * 0.1
    sel = torch.arange(8, dtype=torch.int32, device=gpu).view(1, 1, 1, 8)
    out = c.attend_blocks(q, sel, table, ints([256], gpu))
    ref = c.attend(q, table, ints([256], gpu))
    torch.testing.assert_close(out.float(), ref.float(), rtol=2.0 ** -7, atol=0)


def test_nan_stays_where_it_is_seen(gpu):
    b, d = 1, 64
    k = data(gpu, b, 128, 1, d, BF, 32)
    k[0, 40] = float("nan")
    c, table, _, _, _ = filled(gpu, b, [128], 1, d, 32, BF, 33, k=k)
    q = data(gpu, b, 2, 2, d, BF, 34)
    sel = torch.tensor([[0, 1, -1], [0, 2, 3]], dtype=torch.int32, device=gpu)
    out = c.attend_blocks(q, sel.view(1, 2, 1, 3), table, ints([128], gpu))
    assert torch.isnan(out[0, 0]).all() and not torch.isnan(out[0, 1]).any()


def test_strides_of_queries(gpu):
    b, t, d = 2, 3, 128
    lens = [333, 200]
    c, table, kq, vq, vs = filled(gpu, b, lens, 2, d, 64, BF, 35)
    big = data(gpu, b, t + 2, 13, d + 9, BF, 36)
    for q in (big[:, 1:t + 1, 3:11, :d], big[:, :t, 1:9, 5:d + 5],
              data(gpu, 1, 1, 8, d, BF, 37).expand(b, t, 8, d)):
        kv = ints(lens, gpu, torch.int64)
        sel = c.select_blocks(q, table, kv, None, 6)
        exp = target.select_blocks(
            np64(q), bounds_of(kq, lens, 64, table.shape[1]), lens, [t] * b,
            table.shape[1] * 64, 6, 1, 2)
        np.testing.assert_array_equal(sel.cpu().numpy(), exp)
        out = c.attend_blocks(q, sel, table, kv)
        check_blocks(out, q, sel, kq, vq, vs, lens, [t] * b, BF)


def test_graph_replays(gpu):
    """A step recorded once: append with its bounds, selection, attention."""
    b, t, d = 3, 2, 64
    c, table = make(gpu, b, 1024, 2, d, 64, BF, 38)
    k = data(gpu, b, 600, 2, d, BF, 39)
    c.append(k, k, table, ints([0] * b, gpu))
    q = data(gpu, b, t, 4, d, BF, 40)
    x = k[:, :t].clone()
    start, kv = ints([600] * b, gpu), ints([602] * b, gpu)
    c.select_blocks(q, table, kv, None, 8)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.append(x, x, table, start)
        sel = c.select_blocks(q, table, kv, None, 8)
        out = c.attend_blocks(q, sel, table, kv)
    for i in range(4):
        x.copy_(data(gpu, b, t, 2, d, BF, 50 + i))
        q.copy_(data(gpu, b, t, 4, d, BF, 60 + i))
        start.copy_(ints([600 + 30 * i, 500, 31 * i], gpu))
        kv.copy_(start + t)
        g.replay()
        got = sel.clone(), out.clone()
        again = c.select_blocks(q, table, kv, None, 8)
        assert torch.equal(got[0], again)
        # (row 0 comes to see positions that were never written: NaN)
        torch.testing.assert_close(got[1], c.attend_blocks(q, again, table, kv),
                                   rtol=0, atol=0, equal_nan=True)
        assert not torch.isnan(got[1][1:]).any()


def test_on_another_device(gpu, elsewhere):
    c, table, kq, vq, vs = filled(gpu, 1, [100], 1, 64, 32, BF, 41)
    q = data(gpu, 1, 1, 2, 64, BF, 42)
    kv = ints([100], gpu)
    del elsewhere[:]
    c.update_bounds(table, ints([0], gpu), 100)
    sel = c.select_blocks(q, table, kv, None, 3)
    out = c.attend_blocks(q, sel, table, kv)
    assert elsewhere.count(gpu.index) >= 3
    check_blocks(out, q, sel, kq, vq, vs, [100], [1], BF)


def test_refusals(gpu):
    from suffixgpu_amd import KV4Cache
    from suffixgpu_amd._lib import SuffixGPUError
    c, table, _, _, _ = filled(gpu, 2, [64, 64], 2, 64, 32, BF, 43)
    plain = KV4Cache(4, 2, 64, page_size=32, device=gpu)
    q = data(gpu, 2, 1, 4, 64, BF, 44)
    kv = ints([64, 64], gpu)
    sel = c.select_blocks(q, table, kv, None, 4)
    for bad in (lambda: plain.select_blocks(q, table, kv),
                lambda: plain.update_bounds(table, kv, 1),
                lambda: plain.bounds(table),
                lambda: c.select_blocks(q, table, kv, None, 2),
                lambda: c.select_blocks(q, table, kv, None, 4, -1),
                lambda: c.select_blocks(q, table, kv, None, 4, 1, 0),
                lambda: c.select_blocks(q, table, kv, None, 40000),
                lambda: c.select_blocks(q[:, :, :3], table, kv),
                lambda: c.select_blocks(q.half(), table, kv),
                lambda: c.select_blocks(q, table[:1], kv),
                lambda: c.select_blocks(q, table, kv[:1]),
                lambda: c.attend_blocks(q, sel.long(), table, kv),
                lambda: c.attend_blocks(q, sel[:1], table, kv),
                lambda: c.attend_blocks(q, sel[..., :0], table, kv),
                lambda: c.attend_blocks(q, sel[..., ::2], table, kv),
                lambda: c.attend_blocks(q, sel[:, :, :1], table, kv)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(SuffixGPUError):
        c.attend_blocks(q, sel.cpu(), table, kv)
    # without bounds lists from elsewhere still serve
    plain.attend_blocks(q, sel, table, kv)
    empty = c.select_blocks(q[:0], table[:0], kv[:0])
    assert empty.shape == (0, 1, 2, 64)
