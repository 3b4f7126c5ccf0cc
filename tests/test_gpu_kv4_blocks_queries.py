"""attend_blocks with queries of many magnitudes, and with infinities and NaN."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import target
from tests.test_gpu_kv4 import BF, HF, data, ints, np64
from tests.test_gpu_kv4_blocks import filled

pytestmark = pytest.mark.gpu

def attend(c, q, table, lens, n=6, scale=None):
    gpu = q.device
    kv = ints(lens, gpu)
    sel = c.select_blocks(q, table, kv, None, n)
    return sel, c.attend_blocks(q, sel, table, kv, None, scale)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("kind", ["apart", "large", "small", "tiny", "digits"])
def test_channels_far_apart(gpu, dtype, d, kind):
    """Channels of many magnitudes, the largest of which meet keys of zero; large
    and small queries, with a scale to match."""
    b, t, hq = 2, 3, 4
    lens = [200, 77]
    k = data(gpu, b, 200, 2, d, dtype, 1)
    q = data(gpu, b, t, hq, d, dtype, 2).float()
    scale = None
    if kind == "apart":
        k[..., 5::32] = 0
        q[..., 5::32] = 500.0
        g = torch.Generator().manual_seed(3)
        q *= (2.0 ** -torch.randint(0, 12, (d,), generator=g).float()).to(gpu)
    elif kind == "large":
        # (sums of 256 products with keys below 2^5 are floats: 2^114 2^13 < 2^128)
        assert float(k.abs().max()) < 32
        top = 60000.0 if dtype == HF else 2.0 ** 114
        q *= top / float(q.abs().max())
        scale = 4.0 / top
    elif kind == "small":
        low = 2.0 ** -20 if dtype == HF else 2.0 ** -100
        q *= low
        scale = 0.1 / low
    elif kind == "tiny":      # what the type has below its normal numbers, too
        q *= 2.0 ** -24 if dtype == HF else 2.0 ** -130
        scale = 0.1 * 2.0 ** 22 if dtype == HF else 0.1 * 2.0 ** 120
    else:                     # every digit of the type set
        q = (torch.sign(q) * (2 - 2.0 ** -7 if dtype == BF else 2 - 2.0 ** -10)
             * 2.0 ** -(torch.arange(d, device=gpu) % 6).float())
    q = q.to(dtype)
    c, table, kq, vq, vs = filled(gpu, b, lens, 2, d, 64, dtype, 4, k=k)
    sel, out = attend(c, q, table, lens, scale=scale)
    exp, bound = target.attend_blocks(np64(q), sel.cpu().numpy(), kq, vq, vs,
                                      lens, [t] * b, scale)
    rel, low = target.ulp16(dtype == HF)
    tol = bound + rel * (np.abs(exp) + bound) + low
    err = np.abs(np64(out) - exp)
    assert (err <= tol).all(), (np.argwhere(err > tol)[:5], err.max())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_no_number_stays_in_its_row(gpu, dtype, d):
    b, t, hq = 1, 4, 4
    c, table, _, _, _ = filled(gpu, b, [150], 2, d, 32, dtype, 5)
    q = data(gpu, b, t, hq, d, dtype, 6)
    kv = ints([150], gpu)
    sel = c.select_blocks(q, table, kv, None, 4)
    ref = c.attend_blocks(q, sel, table, kv)
    q[0, 1, 2, d - 1] = float("nan")
    q[0, 2, 0, 7] = float("inf")
    q[0, 3, 3, 40] = -float("inf")
    out = c.attend_blocks(q, sel, table, kv)
    bad = torch.zeros(t, hq, dtype=torch.bool, device=gpu)
    bad[1, 2] = bad[2, 0] = bad[3, 3] = True
    assert torch.isnan(out[0][bad]).all()
    assert torch.equal(out[0][~bad], ref[0][~bad])
