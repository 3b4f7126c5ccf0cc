"""token_logprobs where many logits are equal, or lie together: against the
definition, and that what is masked by a number takes no longer than the rest."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_logprobs import BF, F32, HF, check, data

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("top", [1, 20, 32])
@pytest.mark.parametrize("v,pad", [(20000, 0), (20003, 2), (70001, 1), (700, 3)])
def test_masked_by_the_lowest_value(gpu, dtype, top, v, pad):
    """A row of the type's lowest value but for none, some, or a stretch of the
    logits; rows of one value, of zeros of both signs, of infinities."""
    low = torch.finfo(dtype).min
    x, tok = data(gpu, 8, 2, v, dtype, 3, pad)
    g = torch.Generator().manual_seed(4)
    keep = torch.rand(2, v, generator=g).to(gpu) < 0.001
    x[0][~keep] = low
    x[1] = low
    x[2, :, 300:] = low
    x[3, :, :v - 25] = low
    x[4] = 0.0
    x[4, :, ::3] = -0.0
    x[4, 1, v // 2] = 1.0
    x[5][torch.rand(2, v, generator=g).to(gpu) < 0.5] = float("inf")
    x[6] = -float("inf")
    x[6, :, 40:90] = -1.5
    x[7] = torch.where(keep, 2.0, 1.0).to(dtype)
    t = torch.tensor([1.0, 0.5, 2.0, 1.0, 1.0, 1.0, 0.0, 0.7], device=gpu)
    from suffixgpu_amd import token_logprobs
    check(token_logprobs(x, tok, t, top), x, tok, t, top)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_many_large_ones_in_one_place(gpu, dtype):
    """More than a wave ranks beside each other, where other parts hold little."""
    from suffixgpu_amd import token_logprobs
    v = 30000
    x, tok = data(gpu, 3, 2, v, dtype, 5)
    x[0, :, 4096:4400] += 30.0
    x[1, :, 9000:9016] += 30.0
    x[1, :, 9000 + 2048:9016 + 2048] += 30.0
    x[2, :, 8180:8300] = 20.0
    x[2, 0, 8200:8290] = 21.0
    for top in (1, 24, 32):
        check(token_logprobs(x, tok, None, top), x, tok, None, top)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_few_values(gpu, dtype):
    """Logits of 3, 30 and 300 values, so that lists end within equal ones."""
    from suffixgpu_amd import token_logprobs
    g = torch.Generator().manual_seed(6)
    x = torch.stack([torch.randint(0, n, (2, 50001), generator=g)
                     for n in (3, 30, 300)]).to(dtype).to(gpu) * 0.25
    tok = torch.randint(0, 50001, (3, 2), generator=g,
                        dtype=torch.int32).to(gpu)
    for top in (2, 9, 32):
        check(token_logprobs(x, tok, None, top), x, tok, None, top)
