"""KV4Cache (append, read, attend) against the definitions in 64 bits
(oracle/target.py)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import target

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def make(gpu, b, positions, heads, d, page, dtype, seed, garbage=True):
    """A cache whose pages start as garbage (every float a NaN, every key scale
    a NaN) and a shuffled page table."""
    from suffixgpu_amd import KV4Cache
    width = -(-positions // page)
    c = KV4Cache(b * width, heads, d, page_size=page, dtype=dtype, device=gpu)
    if garbage:
        c.pages.fill_(255)
    g = torch.Generator().manual_seed(seed)
    table = torch.randperm(b * width, generator=g).to(torch.int32)
    return c, table.view(b, width).to(gpu)


def ints(x, gpu, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=gpu)


def np64(t):
    return t.detach().to("cpu", torch.float64).numpy()


def data(gpu, b, t, heads, d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(b, t, heads, d, generator=g)
    x[..., ::17] *= 6.0
    return x.to(dtype).to(gpu)


def filled(gpu, b, lens, heads, d, page, dtype, seed, cap=None):
    """A cache holding lens[i] random tokens in row i, and what it stands
    for."""
    n = max(max(lens), 1)
    c, table = make(gpu, b, cap or n, heads, d, page, dtype, seed)
    k = data(gpu, b, n, heads, d, dtype, seed + 1)
    v = data(gpu, b, n, heads, d, dtype, seed + 2)
    c.append(k, v, table, ints([0] * b, gpu), ints(lens, gpu))
    half = dtype == HF
    kq = target.quantize_k(np64(k), half)
    vq, vs = target.quantize_v(np64(v))
    return c, table, kq, vq, vs


def check_attend(out, q, kq, vq, vs, kv_len, q_len, dtype, scale=None):
    exp, bound = target.attend(np64(q), kq, vq, vs, kv_len, q_len, scale)
    rel, tiny = target.ulp16(dtype == HF)
    err = np.abs(np64(out) - exp)
    tol = bound + rel * (np.abs(exp) + bound) + tiny
    tol = np.where(bound == 0, 0.0, tol)     # rows that see nothing are zeros
    bad = err > tol
    assert not bad.any(), (np.argwhere(bad)[:5], err[bad][:5], tol[bad][:5])


# ------------------------------------------------------------ append, read
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page,t", [(32, 1), (64, 17), (32, 70), (128, 300)])
def test_append_holds_the_rounded_values(gpu, dtype, d, page, t):
    b, heads, cap = 3, 2, 400
    c, table = make(gpu, b, cap, heads, d, page, dtype, 5)
    k = data(gpu, b, t, heads, d, dtype, 6)
    v = data(gpu, b, t, heads, d, dtype, 7)
    start, count = [0, 31, 77], [t, max(0, t - 2), t]
    c.append(k, v, table, ints(start, gpu), ints(count, gpu))
    gk, gv = c.read(table, ints(start, gpu), t, ints(count, gpu))
    ek = target.quantize_k(np64(k), dtype == HF)
    ev, _ = target.quantize_v(np64(v))
    rel, tiny = target.ulp16(dtype == HF)
    for i in range(b):
        n = count[i]
        np.testing.assert_array_equal(np64(gk)[i, :n], ek[i, :n])
        err = np.abs(np64(gv)[i, :n] - ev[i, :n])
        assert (err <= np.abs(ev[i, :n]) * (rel + 2.0 ** -22) + tiny).all()
        assert not np64(gk)[i, n:].any() and not np64(gv)[i, n:].any()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_append_rounds_ties_and_extremes(gpu, dtype):
    """Every magnitude of the type's upper bits in one token or another: ties of
    both scales, subnormals, the largest values, zeros of both signs."""
    d, heads = 128, 1
    top = 65504.0 if dtype == HF else 3.38e38
    rows = []
    for amax in (6.0, 7.0, 7.03125, 8.0, 3.5, 12.0, 1.5, 1e-7, 1e-40, top, 0.0):
        base = torch.arange(d, dtype=torch.float64) / 24.0 * (amax / 5.25)
        base[::2] *= -1
        base[7] = amax
        base[40] = -amax
        rows.append(base.clamp(-amax, amax) if amax else base * 0.0)
    x = torch.stack(rows).to(dtype)[None, :, None].to(gpu)
    t = x.shape[1]
    c, table = make(gpu, 1, t, heads, d, 32, dtype, 8)
    c.append(x, x, table, ints([0], gpu))
    gk, gv = c.read(table, ints([0], gpu), t)
    np.testing.assert_array_equal(np64(gk),
                                  target.quantize_k(np64(x), dtype == HF))
    ev, _ = target.quantize_v(np64(x))
    rel, tiny = target.ulp16(dtype == HF)
    assert (np.abs(np64(gv) - ev)
            <= np.abs(ev) * (rel + 2.0 ** -22) + tiny).all()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_append_values_at_the_midpoints(gpu, dtype):
    """Values on, just below and just above every midpoint between two codes,
    for many largest magnitudes."""
    d, n = 128, 400
    bits = torch.int16
    g = torch.Generator().manual_seed(3)
    top = (torch.rand(n, generator=g) * 3 + 0.5).to(dtype)
    top[:64] = (torch.arange(64) * 3).to(dtype)      # exact ties
    top[0] = 1.0
    x = torch.zeros(n, d, dtype=dtype)
    for i, c in enumerate((1, 3, 5, 7, 10, 14, 20)):
        m = (top.double() * c / 24).to(dtype)
        for j, step in enumerate((-2, -1, 0, 1, 2)):
            y = (m.view(bits) + step).view(dtype)
            x[:, 16 * i + 2 * j] = y
            x[:, 16 * i + 2 * j + 1] = -y
    x[:, 127] = top
    assert (x.abs().amax(dim=1) == top).all()
    x = x[None, :, None].to(gpu)
    c, table = make(gpu, 1, n, 1, d, 64, dtype, 8)
    c.append(x, x, table, ints([0], gpu))
    gk, gv = c.read(table, ints([0], gpu), n)
    np.testing.assert_array_equal(np64(gk),
                                  target.quantize_k(np64(x), dtype == HF))
    ev, _ = target.quantize_v(np64(x))
    rel, tiny = target.ulp16(dtype == HF)
    assert (np.abs(np64(gv) - ev)
            <= np.abs(ev) * (rel + 2.0 ** -22) + tiny).all()


def test_append_infinities_and_nan(gpu):
    """They make their group of a key, or their token's values, NaN, and the
    queries that see them; no other group, token or row."""
    d, heads = 128, 2
    c, table = make(gpu, 1, 64, heads, d, 32, BF, 9)
    k = data(gpu, 1, 40, heads, d, BF, 10)
    v = data(gpu, 1, 40, heads, d, BF, 11)
    k[0, 35, 0, 40] = float("inf")
    v[0, 38, 1, 3] = float("nan")
    c.append(k, v, table, ints([0], gpu))
    gk, gv = c.read(table, ints([0], gpu), 40)
    nk, nv = torch.isnan(gk), torch.isnan(gv)
    assert nk[0, 35, 0, 32:64].all() and int(nk.sum()) == 32
    assert nv[0, 38, 1].all() and int(nv.sum()) == d
    q = data(gpu, 1, 40, heads, d, BF, 12)
    out = c.attend(q, table, ints([40], gpu))
    bad = torch.isnan(out).any(dim=-1)[0]
    assert bad[35:, 0].all() and not bad[:35, 0].any()
    assert bad[38:, 1].all() and not bad[:38, 1].any()


def test_append_keeps_other_tokens_and_overwrites(gpu):
    """Token by token, overlapping and out of order: what is held at the end is
    each position's last write."""
    d, heads, n = 64, 3, 100
    c, table = make(gpu, 2, n, heads, d, 32, BF, 13)
    rng = np.random.default_rng(1)
    want_k = np.zeros((2, n, heads, d))
    want_v = np.zeros((2, n, heads, d))
    c.pages.zero_()
    for step in range(40):
        t = int(rng.integers(1, 9))
        k = data(gpu, 2, t, heads, d, BF, 100 + step)
        v = data(gpu, 2, t, heads, d, BF, 200 + step)
        start = [int(rng.integers(0, n - t + 1)) for _ in range(2)]
        count = [int(rng.integers(0, t + 1)) for _ in range(2)]
        c.append(k, v, table, ints(start, gpu, torch.int64),
                 ints(count, gpu, torch.int64))
        ek = target.quantize_k(np64(k), False)
        ev, _ = target.quantize_v(np64(v))
        for i in range(2):
            want_k[i, start[i]:start[i] + count[i]] = ek[i, :count[i]]
            want_v[i, start[i]:start[i] + count[i]] = ev[i, :count[i]]
    gk, gv = c.read(table, ints([0, 0], gpu), n)
    np.testing.assert_array_equal(np64(gk), want_k)
    err = np.abs(np64(gv) - want_v)
    assert (err <= np.abs(want_v) * (2.0 ** -8 + 2.0 ** -22)).all()


def test_append_outside_the_table_writes_nothing(gpu):
    d, heads = 64, 1
    c, table = make(gpu, 3, 64, heads, d, 32, BF, 14)
    before = c.pages.clone()
    k = data(gpu, 3, 8, heads, d, BF, 15)
    table[1, 1] = -1
    table[2, 1] = c.num_pages
    # past the end, into a page id that is none, and before position 0
    c.append(k, k, table, ints([64, 32, 40], gpu))
    c.append(k, k, table, ints([-1, 1 << 20, -8], gpu))
    assert torch.equal(before, c.pages)
    # only the part inside the table is written and read
    c.append(k, k, table, ints([60, 28, 28], gpu))
    gk, _ = c.read(table, ints([60, 28, 28], gpu), 8)
    ek = target.quantize_k(np64(k), False)
    np.testing.assert_array_equal(np64(gk)[:, :4], ek[:, :4])
    assert not np64(gk)[:, 4:].any()


# ---------------------------------------------------------------- attend
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,heads", [(4, 4), (6, 2), (8, 1)])
@pytest.mark.parametrize("t", [1, 5, 17])
def test_attend_shapes(gpu, dtype, d, hq, heads, t):
    lens = [t, 33, 64, 200]
    lens = [max(x, t) for x in lens]
    c, table, kq, vq, vs = filled(gpu, 4, lens, heads, d, 32, dtype, 20)
    q = data(gpu, 4, t, hq, d, dtype, 21)
    out = c.attend(q, table, ints(lens, gpu))
    check_attend(out, q, kq, vq, vs, lens, [t] * 4, dtype)


@pytest.mark.parametrize("page", [32, 64, 256])
@pytest.mark.parametrize("t", [1, 17])
def test_attend_lengths(gpu, page, t):
    """Rows of no token, one, and around blocks and pages; fewer queries than
    T, none, and more queries than tokens."""
    lens = [0, 1, 2, 31, 32, 33, 63, 65, 257, 700]
    qn = [min(t, max(1, n)) for n in lens]
    qn[4] = 0
    qn[2] = t        # queries before position 0 see nothing
    b = len(lens)
    c, table, kq, vq, vs = filled(gpu, b, lens, 2, 128, page, BF, 30, cap=800)
    q = data(gpu, b, t, 4, 128, BF, 31)
    out = c.attend(q, table, ints(lens, gpu, torch.int64),
                   ints(qn, gpu, torch.int64))
    check_attend(out, q, kq, vq, vs, lens, qn, BF)
    assert not np64(out)[0].any() and not np64(out)[4].any()


@pytest.mark.parametrize("dtype,d,hq,heads", [(BF, 128, 8, 2), (HF, 64, 3, 3),
                                              (HF, 256, 4, 1)])
def test_attend_prompt(gpu, dtype, d, hq, heads):
    """A prompt's chunk of many rows, ragged, after a context."""
    t, lens, qn = 150, [150, 411], [150, 133]
    c, table, kq, vq, vs = filled(gpu, 2, lens, heads, d, 64, dtype, 40)
    q = data(gpu, 2, t, hq, d, dtype, 41)
    out = c.attend(q, table, ints(lens, gpu), ints(qn, gpu))
    check_attend(out, q, kq, vq, vs, lens, qn, dtype)


@pytest.mark.parametrize("t", [1, 3])
def test_attend_long_row_is_split_and_joined(gpu, t):
    lens = [5000, 1300]
    c, table, kq, vq, vs = filled(gpu, 2, lens, 1, 128, 64, BF, 50)
    q = data(gpu, 2, t, 4, 128, BF, 51)
    out = c.attend(q, table, ints(lens, gpu))
    check_attend(out, q, kq, vq, vs, lens, [t] * 2, BF)


@pytest.mark.parametrize("dtype,d", [(BF, 64), (BF, 128), (HF, 128), (HF, 256)])
@pytest.mark.parametrize("t", [1, 17])
def test_attend_splits_of_ragged_rows(gpu, dtype, d, t):
    """Rows of many splits beside rows of one, in tiles of both heights and a
    last tile of a few queries."""
    lens = [4100, 700, t, 2600]
    c, table, kq, vq, vs = filled(gpu, 4, lens, 2, d, 64, dtype, 55)
    q = data(gpu, 4, t, 8, d, dtype, 56)
    out = c.attend(q, table, ints(lens, gpu))
    check_attend(out, q, kq, vq, vs, lens, [t] * 4, dtype)


@pytest.mark.parametrize("scale", [0.0, -0.1, 1e-30, 1e-38, 3.0])
@pytest.mark.parametrize("d,t", [(128, 2), (128, 20), (256, 20)])
def test_attend_any_scale(gpu, d, t, scale):
    """Scales of zero (a mean), below it, next to it and large ones."""
    n = 70
    c, table, kq, vq, vs = filled(gpu, 1, [n], 1, d, 64, BF, 59)
    q = data(gpu, 1, t, 2, d, BF, 60)
    out = c.attend(q, table, ints([n], gpu), scale=scale)
    check_attend(out, q, kq, vq, vs, [n], [t], BF, scale)


@pytest.mark.parametrize("n", [40, 3000])
@pytest.mark.parametrize("t", [2, 20])
def test_attend_nan_queries_say_so(gpu, n, t):
    """A query that holds a NaN gives NaN, in one split or many, and no other
    query does."""
    c, table, *_ = filled(gpu, 1, [n], 1, 128, 64, BF, 57)
    q = data(gpu, 1, t, 2, 128, BF, 58)
    q[0, t - 1, 1, 5] = float("nan")
    bad = torch.isnan(c.attend(q, table, ints([n], gpu)))
    assert bad[0, t - 1, 1].all() and int(bad.sum()) == 128


def test_attend_scales_far_apart(gpu):
    """Values whose scales differ by 2^40 and more, tokens of zero values, a
    large softmax scale: weights stay in range."""
    n, d = 300, 128
    c, table = make(gpu, 1, n, 1, d, 64, BF, 60)
    k = data(gpu, 1, n, 1, d, BF, 61)
    v = data(gpu, 1, n, 1, d, BF, 62)
    g = torch.Generator().manual_seed(63)
    e = torch.randint(-60, 20, (n, 1, 1), generator=g).to(gpu)
    v = torch.ldexp(v[0].float(), e).to(BF)[None]
    v[0, ::13] = 0
    c.append(k, v, table, ints([0], gpu))
    q = data(gpu, 1, 4, 2, d, BF, 64)
    kq = target.quantize_k(np64(k), False)
    vq, vs = target.quantize_v(np64(v))
    for scale in (0.02, 1.0):
        out = c.attend(q, table, ints([n], gpu), scale=scale)
        check_attend(out, q, kq, vq, vs, [n], [4], BF, scale)


def test_attend_strides_and_alignment(gpu):
    """Queries as slices of a fused projection, of misaligned rows, and of
    transposed storage."""
    b, t, hq, d, lens = 2, 7, 4, 64, [90, 40]
    c, table, kq, vq, vs = filled(gpu, b, lens, 2, d, 32, BF, 70)
    fused = data(gpu, b, t, hq + 5, d, BF, 71)
    odd = torch.zeros(b * t * hq * d + 1, dtype=BF, device=gpu)
    odd[1:] = fused[:, :, :hq].reshape(-1)
    qs = [fused[:, :, 1:1 + hq], odd[1:].view(b, t, hq, d),
          fused[:, :, :hq].transpose(1, 2).contiguous().transpose(1, 2)]
    wide = torch.full((b, table.shape[1] + 3), -7, dtype=torch.int32,
                      device=gpu)
    wide[:, :table.shape[1]] = table
    for q in qs:
        out = c.attend(q, wide[:, :table.shape[1]], ints(lens, gpu))
        check_attend(out, q, kq, vq, vs, lens, [t] * b, BF)
    k = data(gpu, b, t, 4, d, BF, 72)
    for src in (k[:, :, 1:3], k[:, :, ::2]):
        c.append(src, src, table, ints([0, 3], gpu))
        gk, _ = c.read(table, ints([0, 3], gpu), t)
        np.testing.assert_array_equal(np64(gk),
                                      target.quantize_k(np64(src), False))
    flat = torch.zeros(k.numel() + 3, dtype=BF, device=gpu)
    flat[3:] = k.reshape(-1)
    src = flat[3:].view(k.shape)[:, :, :2]
    c.append(src, src, table, ints([1, 2], gpu))
    gk, _ = c.read(table, ints([1, 2], gpu), t)
    np.testing.assert_array_equal(np64(gk),
                                  target.quantize_k(np64(src), False))


def test_attend_skips_pages_that_are_none(gpu):
    """A page id that is none hides its positions."""
    c, table, kq, vq, vs = filled(gpu, 2, [96, 96], 1, 64, 32, BF, 80)
    q = data(gpu, 2, 1, 2, 64, BF, 81)
    cut = table.clone()
    cut[0, 1] = -1
    cut[1, 1] = 1 << 30
    out = c.attend(q, cut, ints([96, 96], gpu))
    keep = np.r_[0:32, 64:96]
    check_attend(out, q, kq[:, keep], vq[:, keep], vs[:, keep], [64, 64],
                 [1, 1], BF)
    cut[:] = -1
    assert not np64(c.attend(q, cut, ints([96, 96], gpu))).any()


def test_attend_is_repeatable_and_independent_of_the_batch(gpu):
    lens = [900, 77]
    c, table, *_ = filled(gpu, 2, lens, 2, 128, 64, BF, 90)
    q = data(gpu, 2, 3, 8, 128, BF, 91)
    a = c.attend(q, table, ints(lens, gpu))
    for _ in range(5):
        assert torch.equal(a, c.attend(q, table, ints(lens, gpu)))


def test_cache_under_graph_and_on_another_stream(gpu):
    """append + attend captured and replayed with other data in between, and on
    a side stream."""
    lens = [130, 40]
    c, table, *_ = filled(gpu, 2, lens, 2, 128, 64, BF, 95, cap=200)
    k = data(gpu, 2, 3, 2, 128, BF, 96)
    q = data(gpu, 2, 3, 4, 128, BF, 97)
    start, ln = ints(lens, gpu), ints([n + 3 for n in lens], gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.append(k, k, table, start)
        c.attend(q, table, ln)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.append(k, k, table, start)
        out = c.attend(q, table, ln)
    for seed in (1, 2, 3):
        k.copy_(data(gpu, 2, 3, 2, 128, BF, seed))
        q.copy_(data(gpu, 2, 3, 4, 128, BF, seed + 10))
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        c.append(k, k, table, start)
        assert torch.equal(got, c.attend(q, table, ln))


def test_cache_refusals(gpu):
    from suffixgpu_amd import KV4Cache
    from suffixgpu_amd._lib import SuffixGPUError
    for bad in (dict(head_dim=96), dict(page_size=48), dict(page_size=16),
                dict(dtype=torch.float32), dict(num_kv_heads=0),
                dict(num_pages=-1)):
        with pytest.raises(ValueError):
            KV4Cache(**{**dict(num_pages=4, num_kv_heads=2, head_dim=64,
                               device=gpu), **bad})
    with pytest.raises(SuffixGPUError):
        KV4Cache(4, 2, 64, device="cpu")
    c = KV4Cache(4, 2, 64, page_size=32, device=gpu)
    with pytest.raises(ValueError):
        KV4Cache(4, 2, 64, page_size=32, device=gpu, pages=c.pages[:3])
    table = ints([[0, 1], [2, 3]], gpu)
    k = data(gpu, 2, 3, 2, 64, BF, 1)
    q = data(gpu, 2, 3, 4, 64, BF, 1)
    n = ints([3, 3], gpu)
    for args in ((k.half(), k, table, n), (k, k[:, :2], table, n),
                 (k[..., ::2], k, table, n), (k, k, table.long(), n),
                 (k, k, table[:1], n), (k, k, table, n[:1]),
                 (k, k, table.t(), n), (k[:, :, :1], k, table, n),
                 (k, k, table, None)):
        with pytest.raises(ValueError):
            c.append(*args)
    for args in ((q.half(), table, n), (q[:, :, :3], table, n),
                 (q, table, n[:1]), (q, table, None), (q[0], table, n),
                 (q, table, n, n[:1])):
        with pytest.raises(ValueError):
            c.attend(*args)
    with pytest.raises(SuffixGPUError):
        c.attend(q.cpu(), table, n)
    # nothing to do is no error
    assert c.attend(q[:0], table[:0], n[:0]).shape == (0, 3, 4, 64)
    assert c.attend(q[:, :0], table, n).shape == (2, 0, 4, 64)
    c.append(k[:0], k[:0], table[:0], n[:0])
    empty = torch.empty(2, 0, dtype=torch.int32, device=gpu)
    assert not c.attend(q, empty, n).any()


# ------------------------------------------------ lengths past the ends
@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 256)])
@pytest.mark.parametrize("t,positions", [(1, 64), (10, 64), (17, 3008)])
def test_attend_rows_past_their_table(gpu, dtype, d, t, positions):
    """Tokens past the table hold nothing, but count: the queries of a row
    whose drafts run past its last page stand where kv_len and q_len say."""
    over = [0, 1, 6, 9, t + 3]
    b, page = len(over), 32
    c, table, kq, vq, vs = filled(gpu, b, [positions] * b, 2, d, page, dtype,
                                  200)
    lens = [positions + x for x in over]
    q = data(gpu, b, t, 8, d, dtype, 201)
    out = c.attend(q, table, ints(lens, gpu))
    check_attend(out, q, kq, vq, vs, lens, [t] * b, dtype)
    far = [1 << 40] * b                     # every query past the table
    out = c.attend(q, table, ints(far, gpu, torch.int64))
    check_attend(out, q, kq, vq, vs, [positions + t] * b, [t] * b, dtype)


@pytest.mark.parametrize("t", [1, 4, 20])
def test_attend_more_new_tokens_than_queries(gpu, t):
    """q_len past T: the queries given are the first of the new tokens."""
    lens, qn = [70, 70, 64, 5], [t + 1, t + 30, 1 << 20, t + 2]
    c, table, kq, vq, vs = filled(gpu, 4, lens, 2, 128, 32, BF, 210)
    q = data(gpu, 4, t, 4, 128, BF, 211)
    out = c.attend(q, table, ints(lens, gpu), ints(qn, gpu, torch.int64))
    check_attend(out, q, kq, vq, vs, lens, qn, BF)


# ------------------------------------- NaN and the rows that are no queries
@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("n", [60, 3000])
@pytest.mark.parametrize("t,qn", [(2, 1), (8, 5), (20, 5), (20, 12), (20, 17)])
def test_attend_nan_stays_out_of_padding(gpu, d, n, t, qn):
    """A NaN query, an infinite key early in the row and a NaN value there make
    the queries that see them NaN, and leave zeros from q_len on, in one split or
    many and in tiles of both heights."""
    def run(k=None, v=None, q=None):
        c, table = make(gpu, 1, n, 1, d, 64, BF, 220)
        kk, vv = data(gpu, 1, n, 1, d, BF, 221), data(gpu, 1, n, 1, d, BF, 222)
        qq = data(gpu, 1, t, 2, d, BF, 223)
        for x, at in ((kk, k), (vv, v), (qq, q)):
            if at is not None:
                x[at] = float("inf") if x is kk else float("nan")
        c.append(kk, vv, table, ints([0], gpu))
        out = c.attend(qq, table, ints([n], gpu), ints([qn], gpu))
        assert not np64(out)[0, qn:].any()      # a NaN counts as not zero
        return torch.isnan(out[0, :qn]).all(dim=-1)

    assert not run().any()
    assert run(k=(0, 3, 0, 40)).all()
    assert run(v=(0, 3, 0, 40)).all()
    for r in range(qn):
        bad = run(q=(0, r, 1, 5))
        assert bad[r, 1] and int(bad.sum()) == 1


def test_positions_at_the_end_of_64_bits(gpu):
    """Starts and lengths next to 2^63 lie past the table like any other:
    nothing is read or written there."""
    d, heads, t = 64, 2, 70
    c, table, kq, vq, vs = filled(gpu, 2, [64, 64], heads, d, 32, BF, 260)
    before = c.pages.clone()
    far = ints([(1 << 63) - 1, (1 << 63) - 33], gpu, torch.int64)
    gk, gv = c.read(table, far, t)
    assert not np64(gk).any() and not np64(gv).any()
    k = data(gpu, 2, t, heads, d, BF, 261)
    c.append(k, k, table, far)
    assert torch.equal(before, c.pages)
    q = data(gpu, 2, 3, heads, d, BF, 262)
    check_attend(c.attend(q, table, far), q, kq, vq, vs, [67, 67], [3, 3], BF)
    assert not np64(c.attend(q, table, ints([64, 64], gpu), far)).any()


def test_cache_calls_make_their_device_current(gpu, elsewhere):
    """Launches go to the current device, whichever the tensors' is."""
    lens = [70, 33]
    c, table, kq, vq, vs = filled(gpu, 2, lens, 2, 64, 32, BF, 270)
    assert elsewhere == [0]
    q = data(gpu, 2, 3, 4, 64, BF, 271)
    out = c.attend(q, table, ints(lens, gpu))
    check_attend(out, q, kq, vq, vs, lens, [3, 3], BF)
    gk, _ = c.read(table, ints([0, 0], gpu), 33)
    np.testing.assert_array_equal(np64(gk), kq[:, :33])
    assert elsewhere == [0, 0, 0]


def test_cache_keeps_its_pool(gpu):
    """Calls hold the pool's address, so the pool cannot be exchanged."""
    c, _ = make(gpu, 1, 32, 1, 64, 32, BF, 280)
    with pytest.raises(AttributeError):
        c.pages = torch.zeros_like(c.pages)


# ---------------------------------------------- value scales of any size
@pytest.mark.parametrize("big", [1.0, 1e20, 3e38])
@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("t", [1, 20])
@pytest.mark.parametrize("n,at", [(2, 1), (2, 0), (70, 40), (70, 69),
                                  (300, 200), (3000, 0), (3000, 2999)])
def test_attend_counts_tokens_of_small_values(gpu, n, at, t, d, big):
    """Tokens of equal scores, one of which holds values of `big`, the others
    zeros or values at the least scale: each counts once, whether it shares the
    block, the wave or the split."""
    c, table = make(gpu, 1, n, 1, d, 64, BF, 230)
    k = data(gpu, 1, n, 1, d, BF, 231)
    v = torch.zeros(1, n, 1, d, dtype=BF, device=gpu)
    v[0, ::2] = 2.0 ** -100
    v[0, at] = big
    c.append(k, v, table, ints([0], gpu))
    q = torch.zeros(1, t, 2, d, dtype=BF, device=gpu)
    out = np64(c.attend(q, table, ints([n], gpu)))[0]
    see = np.maximum(np.arange(n - t + 1, n + 1), 0)
    top = float(torch.tensor(big).to(BF))
    want = np.where(see > at, top / np.maximum(see, 1), 0.0)[:, None, None]
    # the value's and the result's rounding, approximations of 1 / s and of
    # exponentials (2^-17); the small values beside it
    tol = want * (2.0 ** -8 + 2.0 ** -15) + 2.0 ** -99
    assert (np.abs(out - want) <= tol).all(), (out[:, 0, 0], want[:, 0, 0])


@pytest.mark.parametrize("t", [1, 20])
@pytest.mark.parametrize("n", [64, 3000])
def test_attend_values_of_every_exponent(gpu, t, n):
    """Values from the least scale to the type's largest side by side, under
    scores that favour one or the other."""
    d = 128
    c, table = make(gpu, 1, n, 1, d, 64, BF, 240)
    k = data(gpu, 1, n, 1, d, BF, 241)
    g = torch.Generator().manual_seed(242)
    e = torch.randint(-104, 122, (1, n, 1, 1), generator=g)
    v = torch.randn(1, n, 1, d, generator=g).clamp(-4, 4)
    v = torch.ldexp(v, e).to(BF).to(gpu)
    c.append(k, v, table, ints([0], gpu))
    q = data(gpu, 1, t, 2, d, BF, 243)
    kq = target.quantize_k(np64(k), False)
    vq, vs = target.quantize_v(np64(v))
    for scale in (0.002, 0.05, 1.0):
        out = c.attend(q, table, ints([n], gpu), scale=scale)
        check_attend(out, q, kq, vq, vs, [n], [t], BF, scale)


@pytest.mark.parametrize("t", [1, 20])
@pytest.mark.parametrize("d,heads", [(64, 1), (128, 2), (256, 1)])
def test_attend_value_scales_of_zero_count(gpu, t, d, heads):
    """Blocks that were never written (zeros throughout) hold keys and values of
    zero: their tokens count in the sum of weights as any other."""
    n, lo = 200, 77
    c, table = make(gpu, 1, n, heads, d, 32, BF, 250)
    c.pages.zero_()
    k = data(gpu, 1, n - lo, heads, d, BF, 251)
    v = data(gpu, 1, n - lo, heads, d, BF, 252)
    c.append(k, v, table, ints([lo], gpu))
    q = data(gpu, 1, t, 2 * heads, d, BF, 253)
    kq = np.zeros((1, n, heads, d))
    vq, vs = np.zeros((1, n, heads, d)), np.ones((1, n, heads, 1))
    kq[:, lo:] = target.quantize_k(np64(k), False)
    vq[:, lo:], vs[:, lo:] = target.quantize_v(np64(v))
    for scale in (0.01, 0.1):
        out = c.attend(q, table, ints([n], gpu), scale=scale)
        check_attend(out, q, kq, vq, vs, [n], [t], BF, scale)
    # a row of nothing else has a mean of zeros
    c.pages.zero_()
    assert not np64(c.attend(q, table, ints([n], gpu))).any()


@pytest.mark.parametrize("t", [1, 17])
def test_attend_many_light_tokens_beside_a_heavy_one(gpu, t):
    """2^18 tokens in one split, one in each wave's share 2^25.1 times as heavy
    as every other: the others are 2^-9 of the sum, and count in the result as
    they do in the sum of weights."""
    from suffixgpu_amd import KV4Cache
    n, d, page, b = 1 << 18, 64, 1 << 16, 1600
    heavy = [0, 32, 64, 96]
    c = KV4Cache(n // page, 1, d, page_size=page, dtype=HF, device=gpu)
    table = torch.arange(n // page, dtype=torch.int32, device=gpu)[None]
    k = torch.zeros(1, n, 1, d, dtype=HF, device=gpu)
    v = torch.full((1, n, 1, d), -1.0, dtype=HF, device=gpu)
    k[0, heavy, 0, 0], v[0, heavy] = 6.0, 1.0
    c.append(k, v, table, ints([0], gpu))
    q = torch.zeros(b, t, 1, d, dtype=HF, device=gpu)
    q[..., 0] = 1.0
    out = c.attend(q, table.expand(b, -1), ints([n], gpu).expand(b),
                   scale=25.1 * np.log(2.0) / 6.0)
    light = np.arange(n - t + 1, n + 1) - len(heavy)
    light = light * 2.0 ** -25.1
    want = ((len(heavy) - light) / (len(heavy) + light))[None, :, None, None]
    # the sum of weights of a lane that begins with a heavy one may lose its
    # light ones (2^15 at most, 2^-10 of it); 2^12 products summed in 32 bits; the
    # result's rounding
    tol = 2.0 ** -10 + 2.0 ** -11 + 2.0 ** -12
    assert (np.abs(np64(out) - want) <= tol).all(), np64(out)[0, :, 0, 0]


@pytest.mark.parametrize("t", [1, 3, 20])
def test_attend_rows_alone_together_and_in_wider_tables(gpu, t):
    """How a row is split follows the call's shape; what it gives does not, up to
    the order of its sums: rows by themselves, among many others, and in tables
    far wider than the rows."""
    lens = [900, 77, 2500]
    c, table, kq, vq, vs = filled(gpu, 3, lens, 2, 128, 64, BF, 290)
    q = data(gpu, 3, t, 8, 128, BF, 291)
    wide = torch.full((3, 20 * table.shape[1]), -1, dtype=torch.int32,
                      device=gpu)
    wide[:, :table.shape[1]] = table
    for tab in (table, wide):
        for i in range(3):
            out = c.attend(q[i:i + 1], tab[i:i + 1], ints(lens[i:i + 1], gpu))
            check_attend(out, q[i:i + 1], kq[i:i + 1], vq[i:i + 1],
                         vs[i:i + 1], lens[i:i + 1], [t], BF)
        many = torch.arange(120, device=gpu) % 3
        out = c.attend(q[many], tab[many], ints(lens, gpu)[many])
        check_attend(out[:3], q, kq, vq, vs, lens, [t] * 3, BF)
        for i in range(3, 120, 3):
            assert torch.equal(out[i:i + 3], out[:3])
