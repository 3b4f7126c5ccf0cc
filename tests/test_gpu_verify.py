"""verify_draft against its definition in 64 bits (oracle/target.py)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import target

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def inputs(gpu, b, k, v, dtype, seed, probs=False, pad=0, agree=0.7,
           temps="mixed"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(b, k + 1, v + pad, generator=g) * 2.5
    draft = torch.randint(0, v, (b, k), generator=g, dtype=torch.int32)
    num = torch.randint(0, k + 1, (b,), generator=g, dtype=torch.int32)
    boost = torch.rand(b, k, generator=g) < agree
    for j in range(k):
        at = draft[:, j].long()
        lift = torch.logsumexp(x[:, j, :v], dim=1) + 3.0
        cur = x[torch.arange(b), j, at]
        x[torch.arange(b), j, at] = torch.where(boost[:, j], lift, cur)
    x = x.to(dtype)
    t = torch.rand(b, generator=g) * 0.8 + 0.5
    if temps == "mixed":
        t[::3] = 0.0
    u = torch.rand(b, k, generator=g)
    e = torch.empty(b, v).exponential_(generator=g)
    q = None
    if probs:
        q = torch.softmax(x[:, :k, :v].float() * 0.8
                          + 0.5 * torch.randn(b, k, v, generator=g), dim=2)
    to = (lambda y: None if y is None else y.to(gpu))
    return dict(logits=to(x)[..., :v], draft=to(draft), num_valid=to(num),
                uniform=to(u), noise=to(e), temperature=to(t),
                draft_probs=to(q))


def oracle(s, greedy=False):
    def a(t):
        return None if t is None else t.float().cpu().numpy()
    t = np.zeros(len(s["num_valid"])) if greedy else a(s["temperature"])
    return target.verify(a(s["logits"]), s["draft"].cpu().numpy(),
                         s["num_valid"].cpu().numpy(), a(s["uniform"]),
                         a(s["noise"]), t, a(s["draft_probs"]))


def check(s, least_clear=0.9, **kw):
    from suffixgpu_amd import verify_draft
    sampled, count = verify_draft(**s, **kw)
    es, ec, clear = oracle(s, kw.get("greedy", False))
    assert clear.mean() >= least_clear, clear.mean()
    np.testing.assert_array_equal(sampled.cpu().numpy()[clear], es[clear])
    np.testing.assert_array_equal(count.cpu().numpy()[clear], ec[clear])
    return sampled, count


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("b,k,v", [(1, 1, 1), (3, 4, 7), (16, 16, 1000),
                                   (9, 5, 8191), (4, 3, 8193),
                                   (2, 7, 40007)])
def test_verify_shapes(gpu, dtype, probs, b, k, v):
    s = inputs(gpu, b, k, v, DTYPES[dtype], b * 1000 + v, probs=probs)
    check(s)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("pad", [1, 3, 8])
def test_verify_strides(gpu, dtype, pad):
    """Logits as a slice of wider rows (rows start at any alignment), and as
    positions spread over a larger buffer."""
    s = inputs(gpu, 6, 5, 8200, DTYPES[dtype], pad, pad=pad)
    check(s)
    x = s["logits"]
    wide = torch.zeros(12, 9, x.shape[2] + pad, dtype=x.dtype, device=gpu)
    wide[::2, 3:, pad:] = x
    s["logits"] = wide[::2, 3:, pad:]
    check(s)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_verify_greedy(gpu, dtype):
    """Ties go to the lowest token; neither random numbers nor temperatures."""
    from suffixgpu_amd import verify_draft
    s = inputs(gpu, 24, 6, 20000, DTYPES[dtype], 3)
    s["logits"].copy_(s["logits"].float().round())   # many equal logits
    top = s["logits"][:, :6].float().argmax(dim=2).int()
    keep = torch.rand(24, 6, generator=torch.Generator().manual_seed(4)) < 0.8
    s["draft"] = torch.where(keep.to(gpu), top, s["draft"])
    got = check(s, least_clear=0.5, greedy=True)
    s["temperature"].zero_()
    again = check(s, least_clear=0.5)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
    bare = verify_draft(s["logits"], s["draft"], s["num_valid"], greedy=True)
    assert torch.equal(got[0], bare[0])


def test_verify_no_drafts_and_all_kept(gpu):
    s = inputs(gpu, 12, 4, 3000, torch.bfloat16, 7, agree=1.0)
    s["uniform"].zero_()
    s["num_valid"].fill_(4)
    s["temperature"].fill_(1.0)
    sampled, count = check(s)
    assert (count == 5).all()
    assert torch.equal(sampled[:, :4], s["draft"])
    s["num_valid"].zero_()
    _, count = check(s)
    assert (count == 1).all()
    # a draft buffer of no columns
    from suffixgpu_amd import verify_draft
    one = verify_draft(s["logits"][:, :1], s["draft"][:, :0].contiguous(),
                       s["num_valid"], s["uniform"][:, :0].contiguous(),
                       s["noise"], s["temperature"])
    again = verify_draft(**s)
    assert torch.equal(one[0], again[0][:, :1])


def test_verify_masked_logits(gpu):
    """-inf, the type's lowest value, NaN and +inf among the logits, a position
    that is all -inf, drafts that are masked."""
    for dtype in DTYPES.values():
        s = inputs(gpu, 20, 4, 9000, dtype, 11)
        x = s["logits"]
        g = torch.Generator().manual_seed(12)
        m = (torch.rand(x.shape, generator=g) < 0.5).to(gpu)
        x[0:4].masked_fill_(m[0:4], float("-inf"))
        x[4:8].masked_fill_(m[4:8], torch.finfo(dtype).min)
        x[8:12].masked_fill_(m[8:12], float("nan"))
        x[12, 0] = float("-inf")
        x[13, 1] = float("nan")
        x[14, 0] = float("-inf")
        x[14, 0, 77] = 1.0              # one candidate
        s["draft"][14, 0] = 77
        x[15, 0] = float("-inf")
        x[15, 0, 8999] = 1.0
        s["draft"][15, 0] = 3
        x[16, 0, 100] = float("inf")
        x[16, 0, 200] = float("inf")    # they share
        s["num_valid"][12:17] = 4
        s["draft"][17, 0] = -1          # ids that are no token end the draft
        s["draft"][18, 1] = 9000
        check(s)


def test_verify_extreme_temperatures(gpu):
    s = inputs(gpu, 8, 3, 5000, torch.float32, 15, temps="all")
    s["temperature"].copy_(torch.tensor([1e-30, 1e-6, 1e-3, 0.05, 20.0, 1e6,
                                         1e30, 1.0]))
    check(s, least_clear=0.5)
    # none or less than none is greedy
    s["temperature"].copy_(torch.tensor([-1.0, float("nan"), 0.0, -0.0, 1.0,
                                         1.0, 1.0, 1.0]))
    check(s, least_clear=0.5)
    s["temperature"] = None
    from suffixgpu_amd import verify_draft
    a = verify_draft(**s)
    s["temperature"] = torch.ones(8, device=gpu)
    b = verify_draft(**s)
    assert torch.equal(a[0], b[0])


@pytest.mark.parametrize("probs", [False, True])
def test_verify_draws_from_the_target(gpu, probs):
    """Whatever is drafted, the first token out is distributed as the target's:
    2^16 rows of one distribution over 6 tokens, against 5 standard
    deviations."""
    from suffixgpu_amd import verify_draft
    n, v, k = 1 << 16, 6, 2
    g = torch.Generator(device=gpu).manual_seed(5)
    x = torch.tensor([2.0, 1.0, 0.0, 0.5, -1.0, 1.5], device=gpu)
    q = torch.tensor([0.05, 0.4, 0.25, 0.1, 0.1, 0.1], device=gpu)
    draft = torch.multinomial(q.expand(n * k, v), 1, generator=g)
    draft = draft.view(n, k).int() if probs else torch.ones(
        n, k, dtype=torch.int32, device=gpu)
    sampled, count = verify_draft(
        x.expand(n, k + 1, v).contiguous(), draft,
        torch.full((n,), k, dtype=torch.int32, device=gpu),
        torch.rand(n, k, generator=g, device=gpu),
        torch.empty(n, v, device=gpu).exponential_(generator=g),
        draft_probs=q.expand(n, k, v).contiguous() if probs else None)
    p = torch.softmax(x.double().cpu(), dim=0)
    first = torch.bincount(sampled[:, 0].long().cpu(), minlength=v) / n
    assert ((first - p).abs() < 5 * (p * (1 - p) / n).sqrt()).all()
    two = sampled[count >= 2][:, 1].long().cpu()
    m = len(two)
    second = torch.bincount(two, minlength=v) / m
    assert ((second - p).abs() < 5 * (p * (1 - p) / m).sqrt()).all()


def test_verify_feeds_the_drafter(gpu):
    """sampled is propose_with_update's sampled_token_ids."""
    from suffixgpu_amd import SuffixGPUDrafter, verify_draft
    d = SuffixGPUDrafter(k=4, device=gpu)
    rows = torch.zeros(3, 64, dtype=torch.int32, device=gpu)
    rows[:, :12] = torch.arange(12, device=gpu).int() % 5
    n = torch.full((3,), 12, dtype=torch.int32, device=gpu)
    draft, nv = d.propose(n, rows)
    x = torch.zeros(3, 5, 50, device=gpu)
    for j in range(4):
        x[:, j].scatter_(1, draft[:, j:j + 1].clamp(min=0).long(), 9.0)
    x[:, 4, 49] = 9.0
    sampled, count = verify_draft(x, draft, nv, greedy=True)
    _, _, new = d.propose_with_update(n, rows, sampled)
    assert torch.equal(new, n + count)
    for i in range(3):
        c = int(count[i])
        assert torch.equal(rows[i, 12:12 + c], sampled[i, :c])


def test_verify_under_graph(gpu):
    from suffixgpu_amd import verify_draft
    s = inputs(gpu, 10, 5, 20011, torch.bfloat16, 21)
    verify_draft(**s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = verify_draft(**s)
    for seed in (31, 32, 33):
        new = inputs(gpu, 10, 5, 20011, torch.bfloat16, seed)
        for name, t in s.items():
            if t is not None:
                t.copy_(new[name])
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        eager = verify_draft(**s)
        assert torch.equal(got[0], eager[0]) and torch.equal(got[1], eager[1])


def test_verify_graphs_of_one_stream_replayed_on_two(gpu):
    """Two graphs recorded by the same stream share nothing: replayed at the
    same time, before and after other calls, each gives its own result, also
    where no call of that size came before the recording."""
    from suffixgpu_amd import verify_draft
    cases = [inputs(gpu, 24, 7, 60013, torch.bfloat16, s) for s in (41, 42)]
    record, graphs, outs = torch.cuda.Stream(), [], []
    for s in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=record):
            outs.append(verify_draft(**s))
        graphs.append(g)
    want = [verify_draft(**s) for s in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(10):
        for pair in outs:
            for t in pair:
                t.fill_(-7)
        for g, st in zip(graphs, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                g.replay()
        for st in streams:
            torch.cuda.current_stream().wait_stream(st)
        again = verify_draft(**cases[0])
        torch.cuda.synchronize()
        for got, exp in zip(outs + [again], want + want[:1]):
            assert torch.equal(got[0], exp[0]) and torch.equal(got[1], exp[1])


def test_verify_refusals(gpu):
    from suffixgpu_amd import verify_draft
    from suffixgpu_amd._lib import SuffixGPUError
    s = inputs(gpu, 2, 3, 100, torch.float32, 1)

    def refuse(exc=ValueError, **kw):
        with pytest.raises(exc):
            verify_draft(**{**s, **kw})
    refuse(logits=s["logits"].double())
    refuse(logits=s["logits"][0])
    refuse(logits=s["logits"].transpose(1, 2).contiguous().transpose(1, 2))
    refuse(draft=s["draft"].long())
    refuse(draft=s["draft"][:, :2])
    refuse(num_valid=s["num_valid"][:1])
    refuse(uniform=None)
    refuse(noise=None)
    refuse(noise=s["noise"][:, :50])
    refuse(noise=s["noise"].t().contiguous().t())
    refuse(temperature=s["temperature"].double())
    refuse(draft_probs=torch.zeros(2, 3, 99, device=gpu))
    refuse(exc=SuffixGPUError, draft=s["draft"].cpu())
    none = verify_draft(s["logits"][:0], s["draft"][:0], s["num_valid"][:0],
                        greedy=True)
    assert none[0].shape == (0, 4) and none[1].shape == (0,)


def test_verify_from_threads_of_one_stream(gpu):
    """Threads that share the default stream each get their own results, of
    sizes that differ."""
    import threading

    from suffixgpu_amd import verify_draft
    cases = [inputs(gpu, 24, 7, 40013, torch.bfloat16, 51),
             inputs(gpu, 40, 3, 9001, torch.float32, 52)]
    want = [verify_draft(**s) for s in cases]
    torch.cuda.synchronize()
    got = [[] for _ in cases]

    def work(i):
        got[i] = [verify_draft(**cases[i]) for _ in range(40)]

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i, exp in enumerate(want):
        assert len(got[i]) == 40
        for a in got[i]:
            assert torch.equal(a[0], exp[0]) and torch.equal(a[1], exp[1])


def test_verify_makes_its_device_current(gpu, elsewhere):
    """Launches go to the current device, whichever the tensors' is."""
    check(inputs(gpu, 6, 4, 3000, torch.bfloat16, 61))
    assert elsewhere == [0]
