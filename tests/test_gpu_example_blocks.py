"""examples/speculative_decode.py with selected blocks, a page pool and the tokens'
log probabilities."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_example import example  # noqa: F401 (fixture)

pytestmark = pytest.mark.gpu


def test_blocks_that_are_all(gpu, example):  # noqa: F811
    """With as many blocks as the rows have, every token is the target's likeliest
    and its log probability the one of a pass over the finished rows, up to what
    bfloat16 activations leave (as for the tokens themselves: 2^-5 of logits of
    size one, which a difference of two has twice)."""
    from suffixgpu_amd import KV4Cache
    b, prompt, new = 4, 32, 64
    rows, steps, lp = example.decode(batch=b, prompt=prompt, new=new, blocks=4,
                                     report=True)
    _, plain = example.decode(batch=b, prompt=prompt, new=new, draft=False,
                              blocks=4)
    assert steps < plain and lp.shape == (b, new)
    model = example.TinyTarget()
    n = prompt + new
    cache = KV4Cache(b * 2, model.kv_heads, model.head_dim, device=gpu)
    table = torch.arange(b * 2, dtype=torch.int32, device=gpu).view(b, 2)
    zero = torch.zeros(b, dtype=torch.int32, device=gpu)
    logits = model.forward(rows, zero, zero + n, cache, table)[:, prompt - 1:-1]
    got = logits.gather(2, rows[:, prompt:].long()[..., None])[..., 0]
    top = logits.max(dim=2).values
    near = 2.0 ** -5 * top.abs().clamp(min=1.0)
    assert (got >= top - near).all()
    exp = got - logits.logsumexp(dim=2)
    assert ((lp - exp).abs() <= 2 * near).all()


def test_few_blocks_run(gpu, example):  # noqa: F811
    rows, _, lp = example.decode(batch=3, prompt=300, new=30, blocks=4,
                                 temperature=0.3, report=True)
    assert rows.shape == (3, 330) and ((rows >= 0) & (rows < 128)).all()
    assert (lp < 0).all() and torch.isfinite(lp).all()
