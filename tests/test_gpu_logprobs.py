"""token_logprobs against the definition in 64 bits (oracle/target.py)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import target

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def np64(t):
    return t.detach().to("cpu", torch.float64).numpy()


def check(got, logits, tokens, temperature, top):
    lp, h, ids, alt, tol = target.logprobs(
        np64(logits), tokens.cpu().numpy(),
        None if temperature is None else temperature.cpu().numpy(), top)
    for name, x, y, t in (("logprob", got[0], lp, tol[0]),
                          ("entropy", got[1], h, tol[1]),
                          ("top", got[3], alt, tol[2])):
        x = np64(x)
        # what float32 cannot hold is an infinity there
        y = np.where(np.abs(y) >= 2.0 ** 128 - 2.0 ** 103,
                     np.copysign(np.inf, y), y)
        with np.errstate(invalid="ignore"):
            bad = ~((np.abs(x - y) <= t) | (x == y))
        assert not bad.any(), (name, np.argwhere(bad)[:5], x[bad][:5],
                               y[bad][:5], t[bad][:5])
    np.testing.assert_array_equal(got[2].cpu().numpy(), ids)


def data(gpu, b, j, v, dtype, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(b, j, v + pad, generator=g) * 2.5).to(dtype).to(gpu)
    tok = torch.randint(0, v, (b, j), generator=g, dtype=torch.int32)
    return x[..., :v], tok.to(gpu)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("v,pad,top", [
    (1, 0, 1), (2, 3, 5), (7, 1, 7), (33, 0, 32), (1000, 1, 0), (8191, 0, 3),
    (8192, 0, 20), (8193, 7, 32), (32001, 0, 8), (65003, 5, 1)])
def test_sizes_and_alignments(gpu, dtype, v, pad, top):
    from suffixgpu_amd import token_logprobs
    x, tok = data(gpu, 3, 4, v, dtype, v + top, pad)
    tok[0, 2] = -1
    tok[1, 3] = v
    temp = torch.tensor([1.0, 0.0, 0.3], device=gpu)
    got = token_logprobs(x, tok, temp, top)
    assert [tuple(t.shape) for t in got] == [(3, 4), (3, 4), (3, 4, top),
                                             (3, 4, top)]
    check(got, x, tok, temp, top)
    check(token_logprobs(x, tok, top=top), x, tok, None, top)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_likely_tokens_keep_small_logprobs(gpu, dtype):
    """p of the token from 1 - 2^-30 to 2^-3: what the others add to one."""
    from suffixgpu_amd import token_logprobs
    b, v = 24, 20000
    x, _ = data(gpu, b, 1, v, dtype, 1)
    tok = torch.arange(b, device=gpu, dtype=torch.int32)[:, None] * 811
    big = torch.linspace(10, 40, b, device=gpu)[:, None, None].to(dtype)
    x.scatter_(2, tok.long()[..., None], big)
    check(token_logprobs(x, tok, top=4), x, tok, None, 4)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_ties_give_the_lowest(gpu, dtype):
    """All equal, few values, and the largest many times: past what is ranked at
    once, across pieces, vectors and workgroups."""
    from suffixgpu_amd import token_logprobs
    v, top = 20011, 32
    x, tok = data(gpu, 6, 1, v, dtype, 2)
    x[0] = 0.0
    x[1] = x[1].round()
    x[2, 0, ::3] = 9.0
    x[3, 0, -40:] = 9.0
    x[4] = -0.0
    x[4, 0, 5::7] = 0.0
    x[5, 0, 100:140] = 9.0
    x[5, 0, 9000] = 10.0
    for temp in (None, torch.tensor([1, 1, 0, 0, 1, 0.5], device=gpu)):
        check(token_logprobs(x, tok, temp, top), x, tok, temp, top)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_infinities_and_nan(gpu, dtype):
    from suffixgpu_amd import token_logprobs
    v, top = 9001, 6
    inf = float("inf")
    x, tok = data(gpu, 8, 2, v, dtype, 3)
    x[0] = -inf
    x[1] = float("nan")
    x[2, :, 1:] = -inf
    x[3, :, ::2] = -inf
    x[4, :, 17] = inf
    x[5, :, 8999:] = inf
    x[6, :, ::5] = float("nan")
    x[7, :, 4:] = -inf
    x[7, 1, 3] = float("nan")
    tok[2, 0] = 0
    tok[4, 0], tok[4, 1] = 17, 18
    tok[5, 0] = 9000
    tok[6, 0] = 5
    for temp in (None, torch.tensor([0, 1, 0, 1e-30, 1, 0.1, 3, 0.7],
                                    device=gpu)):
        check(token_logprobs(x, tok, temp, top), x, tok, temp, top)


def test_extreme_logits(gpu):
    from suffixgpu_amd import token_logprobs
    x, tok = data(gpu, 4, 1, 9000, F32, 4)
    x[0] *= 1e38
    x[1] *= 1e-38
    x[2, 0, 5] = 3.4e38
    x[3, 0] = 3e38
    x[3, 0, 77] = -3e38
    tok[2] = 5
    for temp in (None, torch.tensor([1e-3, 1e3, 1e-30, 1e30], device=gpu),
                 torch.tensor([3e38, 1e-38, 1e38, 2e38], device=gpu)):
        check(token_logprobs(x, tok, temp, 9), x, tok, temp, 9)


def test_strides(gpu):
    from suffixgpu_amd import token_logprobs
    x, tok = data(gpu, 4, 6, 5003, BF, 5)
    for y, t in ((x[::2, 1::2], tok[::2, 1::2].contiguous()),
                 (x.transpose(0, 1), tok.t().contiguous()),
                 (x[:1].expand(5, 6, 5003), tok[:1].expand(5, 6).contiguous())):
        check(token_logprobs(y, t, top=3), y, t, None, 3)
    one = torch.randn(3, 2, 1, device=gpu)
    got = token_logprobs(one, torch.zeros(3, 2, dtype=torch.int32,
                                          device=gpu), top=2)
    assert (got.logprob == 0).all() and (got.entropy == 0).all()
    assert (got.top_tokens == torch.tensor([0, -1], device=gpu)).all()


def test_empty(gpu):
    from suffixgpu_amd import token_logprobs
    for b, j in ((0, 3), (3, 0)):
        got = token_logprobs(torch.empty(b, j, 10, device=gpu),
                             torch.empty(b, j, dtype=torch.int32, device=gpu),
                             top=2)
        assert got.top_tokens.shape == (b, j, 2)


def test_takes_what_verify_draft_gives(gpu):
    """sampled, its -1 among it: as many positions as count are read."""
    from suffixgpu_amd import token_logprobs, verify_draft
    b, k, v = 5, 4, 3001
    x, tok = data(gpu, b, k + 1, v, BF, 6)
    draft = x[:, :k].float().argmax(dim=2).int()
    draft[1, 2] = (draft[1, 2] + 1) % v
    sampled, count = verify_draft(x, draft, torch.full(
        (b,), k, dtype=torch.int32, device=gpu), greedy=True)
    got = token_logprobs(x, sampled, top=2)
    check(got, x, sampled, None, 2)
    kept = torch.arange(k + 1, device=gpu) < count[:, None]
    assert (got.logprob[kept] < 0).all() and (got.logprob[~kept] == 0).all()
    torch.testing.assert_close(got.top_tokens[..., 0][kept], sampled[kept])


def test_graph_replays(gpu):
    from suffixgpu_amd import token_logprobs
    x, tok = data(gpu, 3, 2, 30011, BF, 7)
    token_logprobs(x, tok, top=5)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = token_logprobs(x, tok, top=5)
    for seed in (8, 9, 10):
        y, t = data(gpu, 3, 2, 30011, BF, seed)
        x.copy_(y)
        tok.copy_(t)
        g.replay()
        again = token_logprobs(x, tok, top=5)
        torch.cuda.synchronize()
        for a, b in zip(out, again):
            assert torch.equal(a, b)
        check(out, x, tok, None, 5)


def test_on_another_device(gpu, elsewhere):
    from suffixgpu_amd import token_logprobs
    x, tok = data(gpu, 2, 2, 9999, BF, 11)
    got = token_logprobs(x, tok, top=3)
    assert gpu.index in elsewhere
    check(got, x, tok, None, 3)


def test_on_another_stream(gpu):
    from suffixgpu_amd import token_logprobs
    x, tok = data(gpu, 2, 2, 9999, BF, 11)
    s = torch.cuda.Stream(device=gpu)
    s.wait_stream(torch.cuda.default_stream(gpu))
    with torch.cuda.stream(s):
        got = token_logprobs(x, tok, top=3)
    s.synchronize()
    check(got, x, tok, None, 3)


def test_refusals(gpu):
    from suffixgpu_amd import token_logprobs
    from suffixgpu_amd._lib import SuffixGPUError
    x, tok = data(gpu, 2, 3, 100, BF, 12)
    temp = torch.ones(2, device=gpu)
    for bad in (lambda: token_logprobs(x[0], tok),
                lambda: token_logprobs(x.double(), tok),
                lambda: token_logprobs(x[..., ::2], tok),
                lambda: token_logprobs(x, tok.long()),
                lambda: token_logprobs(x, tok[:, :2]),
                lambda: token_logprobs(x, tok.t().contiguous().t()),
                lambda: token_logprobs(x, tok, temp[:1]),
                lambda: token_logprobs(x, tok, temp.double()),
                lambda: token_logprobs(x, tok, top=33),
                lambda: token_logprobs(x, tok, top=-1),
                lambda: token_logprobs(x[..., :0], tok),
                lambda: token_logprobs(
                    x.float().requires_grad_(), tok)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(SuffixGPUError):
        token_logprobs(x, tok.cpu())
    with torch.no_grad():
        token_logprobs(x.float().requires_grad_(), tok)
