"""token_logprobs where logits over temperature are large: low temperatures, large
logits, and the least differences that there are between them."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import target
from tests.test_gpu_logprobs import BF, F32, HF, data, np64

pytestmark = pytest.mark.gpu

# What float32 loses at the end of its range, where the definition's 64 bits go on: a
# power below 2^-126 may be zero, and so may its product with z.  In nats |z e^z| is at
# most 88 * 2^-126 there, e^z itself less; of 9,001 < 2^14 logits that is less than
# 2^(14 + 7 - 126), and so is what each of the sums, and log1p of the first, is off by.
LOST = 2.0 ** -105


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
            bad = ~((np.abs(x - y) <= t + LOST) | (x == y))
        assert not bad.any(), (name, np.argwhere(bad)[:5], x[bad][:5],
                               y[bad][:5], t[bad][:5])
    np.testing.assert_array_equal(got[2].cpu().numpy(), ids)


@pytest.mark.parametrize("top", [0, 4])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_low_temperatures(gpu, dtype, top):
    """From 10^-3 to 10^-19; a row for each, several positions as the rounding of the
    largest logit's exponent differs."""
    from suffixgpu_amd import token_logprobs
    temp = torch.tensor([10.0 ** -(3 + i / 2) for i in range(33)], device=gpu)
    x, tok = data(gpu, 33, 6, 3001, dtype, 1)
    x[:, ::2] += x[:, ::2].abs().amax(dim=2, keepdim=True) + 9
    tok[:, 1:4] = x[:, 1:4].float().argmax(dim=2).int()
    check(token_logprobs(x, tok, temp, top), x, tok, temp, top)


@pytest.mark.parametrize("top", [0, 3])
def test_large_logits(gpu, top):
    from suffixgpu_amd import token_logprobs
    x, tok = data(gpu, 36, 4, 9001, F32, 2)
    x *= torch.tensor([10.0 ** i for i in range(36)], device=gpu)[:, None, None]
    tok[:, ::2] = x[:, ::2].argmax(dim=2).int()
    check(token_logprobs(x, tok, None, top), x, tok, None, top)
    # all of them below zero
    y = -x.abs() - x.abs().amax(dim=2, keepdim=True)
    tok[:, ::2] = y[:, ::2].argmax(dim=2).int()
    check(token_logprobs(y, tok, None, top), y, tok, None, top)


@pytest.mark.parametrize("sign", [1, -1])
def test_logits_next_to_the_largest(gpu, sign):
    """The largest and the float below it, a few of each, at temperatures where the
    other is far, near, and as good as equal."""
    from suffixgpu_amd import token_logprobs
    tops = [1.0, 1.7, 3.1, 30.0, 1000.3, 5e6, 1.6777215e7, 3e9, 7e20]
    rows = []
    for t in tops:
        a = torch.tensor(sign * t, dtype=torch.float32)
        b = torch.nextafter(a, torch.tensor(-float("inf")))
        row = torch.full((9001,), float(a - abs(a) * 0.5))
        row[7] = a
        row[100:103] = b
        row[8990] = b
        rows += [(row, float(a - b) * s) for s in (0.05, 0.5, 2.0, 30.0)]
    x = torch.stack([r for r, _ in rows])[:, None].to(gpu)
    temp = torch.tensor([t for _, t in rows], device=gpu)
    tok = torch.full((len(rows), 1), 101, dtype=torch.int32, device=gpu)
    check(token_logprobs(x, tok, temp, 5), x, tok, temp, 5)
