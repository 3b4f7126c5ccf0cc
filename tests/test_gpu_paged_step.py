"""A serving step as one run: PagePool, KV4Cache with bounds, selection, attention
over it, verify_draft and token_logprobs, against the oracle's definitions, eager
and recorded; and calls of theirs at the edges of what they take."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import target
from tests.test_gpu_kv4 import BF, HF, data, ints, np64
from tests.test_gpu_kv4_blocks import bounds_of, check_blocks, filled, make
from tests.test_gpu_logprobs import check as check_logprobs

pytestmark = pytest.mark.gpu

B, HEADS, GROUP, D, PAGE, WIDTH, K, V = 3, 2, 2, 64, 32, 8, 4, 300


class Rows:
    """Three requests' pool, cache and inputs; `step` is what an engine does."""

    def __init__(self, gpu):
        from suffixgpu_amd import KV4Cache, PagePool
        self.pool = PagePool(20, B, WIDTH, page_size=PAGE, device=gpu)
        self.cache = KV4Cache(20, HEADS, D, page_size=PAGE, device=gpu,
                              bounds=True)
        self.cache.pages.fill_(255)
        self.len = torch.zeros(B, dtype=torch.int32, device=gpu)
        self.k = data(gpu, B, K + 1, HEADS, D, BF, 1)
        self.v = data(gpu, B, K + 1, HEADS, D, BF, 2)
        self.q = data(gpu, B, K + 1, HEADS * GROUP, D, BF, 3)
        self.logits = torch.zeros(B, K + 1, V, dtype=BF, device=gpu)
        self.draft = torch.zeros(B, K, dtype=torch.int32, device=gpu)
        self.valid = torch.zeros(B, dtype=torch.int32, device=gpu)
        self.temp = torch.tensor([1.0, 0.5, 0.0], device=gpu)

    def prompt(self, k, v, lens):
        self.pool.resize(lens)
        self.cache.append(k, v, self.pool.table,
                          torch.zeros_like(self.len), lens)
        self.len.copy_(lens)

    def step(self):
        from suffixgpu_amd import token_logprobs, verify_draft
        end = self.len + K + 1
        room = self.pool.resize(end)
        table = self.pool.table
        self.cache.append(self.k, self.v, table, self.len)
        sel = self.cache.select_blocks(self.q, table, end, None, 4)
        out = self.cache.attend_blocks(self.q, sel, table, end)
        sampled, count = verify_draft(self.logits, self.draft, self.valid,
                                      greedy=True)
        lp = token_logprobs(self.logits, sampled, self.temp, 3)
        self.len.add_(count)
        self.pool.resize(self.len)
        return room, sel, out, sampled, count, *lp

    def inputs(self, seed):
        gpu = self.len.device
        g = torch.Generator().manual_seed(seed)
        self.k.copy_(data(gpu, B, K + 1, HEADS, D, BF, 10 * seed))
        self.v.copy_(data(gpu, B, K + 1, HEADS, D, BF, 10 * seed + 1))
        self.q.copy_(data(gpu, B, K + 1, HEADS * GROUP, D, BF, 10 * seed + 2))
        logits = torch.randn(B, K + 1, V, generator=g).to(BF)
        self.logits.copy_(logits)
        draft = logits.argmax(dim=2)[:, :K].to(torch.int32)
        for i in range(B):      # rows differ in how many drafts stay
            draft[i, (seed + i) % (K + 1):] = 0
        self.draft.copy_(draft)
        self.valid.copy_(torch.tensor([K, K - 1, seed % (K + 1)],
                                      dtype=torch.int32))


def prompt_of(gpu):
    return data(gpu, B, 110, HEADS, D, BF, 4), data(gpu, B, 110, HEADS, D, BF,
                                                    5)


def test_steps_are_the_definitions(gpu):
    r = Rows(gpu)
    o = target.Pages(20, B, WIDTH, PAGE)
    pk, pv = prompt_of(gpu)
    lens = [110, 33, 64]
    r.prompt(pk, pv, ints(lens, gpu))
    o.resize(lens)
    hold = [[np64(x)[i, :n] for x in (pk, pv)] for i, n in enumerate(lens)]
    for s in range(6):
        if s == 3:      # one request ends, another takes its place and pages
            lens[0] = 0
            r.len[0] = 0
            hold[0] = [h[:0] for h in hold[0]]
        r.inputs(s + 1)
        room, sel, out, sampled, count, *lp = r.step()
        end = [n + K + 1 for n in lens]
        assert room.tolist() == o.resize(end)
        for i in range(B):
            hold[i] = [np.concatenate([h, np64(x)[i]])
                       for h, x in zip(hold[i], (r.k, r.v))]
        k, v = (np.zeros((B, WIDTH * PAGE, HEADS, D)) for _ in range(2))
        for i in range(B):
            k[i, :end[i]], v[i, :end[i]] = hold[i]
        kq = target.quantize_k(k, False)
        vq, vs = target.quantize_v(v)
        ql = [K + 1] * B
        exp = target.select_blocks(np64(r.q), bounds_of(kq, end, PAGE, WIDTH),
                                   end, ql, WIDTH * PAGE, 4, 1, 2)
        np.testing.assert_array_equal(sel.cpu().numpy(), exp)
        check_blocks(out, r.q, sel, kq, vq, vs, end, ql, BF)
        es, ec, _ = target.verify(np64(r.logits), r.draft.cpu().numpy(),
                                  r.valid.cpu().numpy(), None, None,
                                  np.zeros(B))
        np.testing.assert_array_equal(sampled.cpu().numpy(), es)
        np.testing.assert_array_equal(count.cpu().numpy(), ec)
        check_logprobs(lp, r.logits, sampled, r.temp, 3)
        lens = [n + int(c) for n, c in zip(lens, count)]
        hold = [[x[:n] for x in h] for h, n in zip(hold, lens)]
        o.resize(lens)
        np.testing.assert_array_equal(r.pool.table.cpu().numpy(), o.table())
        assert r.pool.num_free.tolist() == [len(o.free)]


def test_a_recorded_step_is_the_eager_one(gpu):
    one, two = Rows(gpu), Rows(gpu)
    pk, pv = prompt_of(gpu)
    for r in (one, two):
        r.prompt(pk, pv, ints([100, 1, 0], gpu))
        r.inputs(50)
        r.step()                # (both have run once, the recorded one eagerly)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = one.step()
    for s in range(6):
        one.inputs(60 + s)
        two.inputs(60 + s)
        graph.replay()
        exp = two.step()
        for x, y in zip(got, exp):
            torch.testing.assert_close(x, y, rtol=0, atol=0)
        for x, y in ((one.len, two.len), (one.pool.table, two.pool.table),
                     (one.pool.num_free, two.pool.num_free),
                     (one.cache.pages, two.cache.pages)):
            assert torch.equal(x, y)
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d,heads,group,t,n", [
    (64, 1, 1, 16, 3), (64, 1, 12, 3, 5), (128, 2, 17, 4, 6), (128, 1, 2, 8, 1),
    (256, 2, 5, 3, 40), (64, 1, 3, 100, 9)])
@pytest.mark.parametrize("scale", [0.0, -0.1, 1.5])
def test_head_groups_and_scales(gpu, dtype, d, heads, group, t, n, scale):
    """Tiles that a token's heads do not fill, share or pass; scales of any
    sign."""
    lens = [290, 128]
    c, table, kq, vq, vs = filled(gpu, 2, lens, heads, d, 32, dtype, 70 + n)
    q = data(gpu, 2, t, heads * group, d, dtype, 71)
    kv = ints(lens, gpu)
    sel = c.select_blocks(q, table, kv, None, n, 0, 1)
    out = c.attend_blocks(q, sel, table, kv, None, scale)
    check_blocks(out, q, sel, kq, vq, vs, lens, [t] * 2, dtype, scale)
    assert torch.equal(out, c.attend_blocks(q, sel, table, kv, None, scale))


@pytest.mark.parametrize("t,group", [(1, 4), (3, 2), (2, 20)])
def test_lengths_far_past_the_table(gpu, t, group):
    """Where a query stands is kv_len - q_len, whatever these are."""
    c, table, kq, vq, vs = filled(gpu, 2, [150, 90], 1, 64, 32, BF, 72)
    q = data(gpu, 2, t, group, 64, BF, 73)
    lens = [150, 90]
    near = (ints(lens, gpu, torch.int64), ints([t, t], gpu, torch.int64))
    sel = c.select_blocks(q, table, near[0], near[1], 3, 0, 1)
    out = c.attend_blocks(q, sel, table, *near)
    check_blocks(out, q, sel, kq, vq, vs, lens, [t] * 2, BF)
    # (the same queries as the first t of a row's 2^62 and more)
    big = 2 ** 62
    far = (near[0] + big, near[1] + big)
    assert torch.equal(c.select_blocks(q, table, *far, 3, 0, 1), sel)
    assert torch.equal(c.attend_blocks(q, sel, table, *far), out)


def test_tables_and_pools_of_nothing(gpu):
    from suffixgpu_amd import KV4Cache, PagePool
    q = data(gpu, 2, 3, 4, 64, BF, 80)
    kv = ints([3, 70], gpu)
    for c, table in (
            (make(gpu, 2, 96, 2, 64, 32, BF, 81)[0],
             torch.zeros(2, 0, dtype=torch.int32, device=gpu)),
            (KV4Cache(0, 2, 64, page_size=32, device=gpu, bounds=True),
             torch.zeros(2, 3, dtype=torch.int32, device=gpu))):
        k = q[:, :, :2]
        c.append(k, k, table, ints([0, 0], gpu))
        c.update_bounds(table, ints([0, 0], gpu), 100)
        sel = c.select_blocks(q, table, kv, None, 5)
        if table.shape[1] == 0:
            assert (sel == -1).all()
        out = c.attend_blocks(q, sel, table, kv)
        assert out.shape == q.shape and (out == 0).all()
        lo, hi = c.bounds(table)
        assert lo.shape == hi.shape == (2, table.shape[1], 2, 64)
        assert not lo.any() and not hi.any()
    pool = PagePool(0, 2, 3, device=gpu)
    assert pool.resize(ints([64, 1], gpu)).tolist() == [0, 0]
    assert (pool.table == -1).all() and pool.held.tolist() == [0, 0]
    assert (pool.slots(ints([0, 5], gpu), 4) == -1).all()
    assert pool.resize(ints([], gpu)).shape == (0,)
    assert pool.slots(ints([], gpu), 4).shape == (0, 4)
    assert pool.slots(ints([0, 5], gpu), 0).shape == (2, 0)


def test_calls_side_by_side(gpu):
    """The same calls on four streams at once, each with what it needs of its
    own, give what each gives alone."""
    from suffixgpu_amd import token_logprobs
    c, table, _, _, _ = filled(gpu, 2, [3000, 2000], 1, 64, 64, BF, 82)
    kv = ints([3000, 2000], gpu)
    wide = torch.full((2, 1100), -1, dtype=torch.int32, device=gpu)
    wide[:, :table.shape[1]] = table
    x = torch.randn(4, 6, 40000, device=gpu)
    tok = x.argmax(dim=2).to(torch.int32)
    q = data(gpu, 8, 2, 3, 64, BF, 83).view(4, 2, 2, 3, 64)

    def run(i):
        sel = c.select_blocks(q[i], wide, kv, None, 40)
        return (sel, c.attend_blocks(q[i], sel, wide, kv),
                *token_logprobs(x[i:i + 1], tok[i:i + 1], None, 5))

    alone = [run(i) for i in range(4)]
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(run(i))
        torch.cuda.synchronize()
        for a, g in zip(alone, got):
            for y, z in zip(a, g):
                assert torch.equal(y, z)


def test_bounds_refusals(gpu):
    c, table = make(gpu, 2, 64, 2, 64, 32, BF, 84)
    zero = ints([0, 0], gpu)
    for bad in (lambda: c.update_bounds(table.long(), zero, 1),
                lambda: c.update_bounds(table, zero[:1], 1),
                lambda: c.update_bounds(table, zero, 1, zero[:1])):
        with pytest.raises(ValueError):
            bad()
    from suffixgpu_amd._lib import SuffixGPUError
    with pytest.raises(SuffixGPUError):
        c.update_bounds(table, zero, -1)
