"""examples/speculative_decode.py: drafter, 4-bit cache, attention and
verification in one loop."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = Path(__file__).resolve().parents[1] / "examples" / \
    "speculative_decode.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("speculative_decode", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_greedy_tokens_are_the_targets(gpu, example):
    """Every token decoded with drafts is the target's likeliest after the
    tokens before it, as one pass over the finished rows sees it (up to what
    bfloat16 activations leave of logits of size one)."""
    from suffixgpu_amd import KV4Cache
    b, prompt, new = 4, 32, 64
    rows, steps = example.decode(batch=b, prompt=prompt, new=new)
    _, plain = example.decode(batch=b, prompt=prompt, new=new, draft=False)
    assert steps < plain
    model = example.TinyTarget()
    n = prompt + new
    cache = KV4Cache(b * 2, model.kv_heads, model.head_dim, device=gpu)
    table = torch.arange(b * 2, dtype=torch.int32, device=gpu).view(b, 2)
    zero = torch.zeros(b, dtype=torch.int32, device=gpu)
    logits = model.forward(rows, zero, zero + n, cache, table)[:, prompt - 1:-1]
    got = logits.gather(2, rows[:, prompt:].long()[..., None])[..., 0]
    top = logits.max(dim=2).values
    assert (got >= top - 2.0 ** -5 * top.abs().clamp(min=1.0)).all()


def test_sampled_rows_are_full(gpu, example):
    rows, steps = example.decode(batch=3, prompt=20, new=40, temperature=0.3)
    assert rows.shape == (3, 60) and steps >= 1
    assert ((rows >= 0) & (rows < 128)).all()
