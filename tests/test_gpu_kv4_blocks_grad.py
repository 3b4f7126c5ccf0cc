"""attend_blocks and token_logprobs serve a model: what asks for a gradient is refused
rather than answered without one."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_kv4 import BF, data, ints
from tests.test_gpu_kv4_blocks import filled

pytestmark = pytest.mark.gpu


def test_queries_that_ask_for_a_gradient_are_refused(gpu):
    c, table, _, _, _ = filled(gpu, 1, [100], 2, 64, 32, BF, 1)
    q = data(gpu, 1, 2, 4, 64, BF, 2)
    kv = ints([100], gpu)
    sel = c.select_blocks(q, table, kv, None, 3)
    plain = c.attend_blocks(q, sel, table, kv)
    asks = q.clone().requires_grad_()
    with pytest.raises(ValueError, match="detach"):
        c.attend_blocks(asks, sel, table, kv)
    with pytest.raises(ValueError, match="detach"):
        c.attend_blocks(asks * 2, sel, table, kv)
    # a choice of blocks has none, and without a graph there is nothing to lose
    assert torch.equal(c.select_blocks(asks, table, kv, None, 3), sel)
    with torch.no_grad():
        assert torch.equal(c.attend_blocks(asks, sel, table, kv), plain)
    with torch.inference_mode():
        assert torch.equal(c.attend_blocks(asks, sel, table, kv), plain)
    assert torch.equal(c.attend_blocks(asks.detach(), sel, table, kv), plain)


def test_temperatures_that_ask_for_a_gradient_are_refused(gpu):
    from suffixgpu_amd import token_logprobs
    x = torch.randn(2, 3, 100, device=gpu)
    tok = torch.zeros(2, 3, dtype=torch.int32, device=gpu)
    temp = torch.full((2,), 0.7, device=gpu, requires_grad=True)
    with pytest.raises(ValueError, match="detach"):
        token_logprobs(x, tok, temp)
    with torch.no_grad():
        a = token_logprobs(x, tok, temp)
    for y, z in zip(a, token_logprobs(x, tok, temp.detach())):
        assert torch.equal(y, z)
