"""Registers and scratch of the target-side kernels, from the compiler's
resource report.

The attention kernels keep a block of the cache, the queries' operands and the
sums in registers, close below what lets the waves of a SIMD that they are laid
out for stay on it (__launch_bounds__): a few more would go to scratch memory, in
the loop over the cache, without a word."""

from __future__ import annotations

import os
import shutil

import pytest

from suffixgpu_amd import build
from tests.test_kernel_resources import _resources

needs_hipcc = pytest.mark.skipif(
    shutil.which(build.HIPCC) is None and not os.path.exists(build.HIPCC),
    reason="needs hipcc")


def _check(res, kernel, waves):
    found = {k: v for k, v in res.items() if kernel in k}
    assert found, f"no {kernel} in the resource report"
    for name, r in found.items():
        assert r["ScratchSize"] == 0, (name, r)
        assert r["Occupancy"] >= waves, (name, r)


@needs_hipcc
def test_attention_kernels_keep_their_waves(tmp_path):
    res = _resources("kv4_attend.hip", tmp_path)
    # by head size, which the mangled name has as the first argument
    for d, w16, w32 in ((64, 4, 3), (128, 4, 3), (256, 2, 2)):
        _check(res, f"k_kv4_attend16ILi{d}E", w16)
        _check(res, f"k_kv4_attend32ILi{d}E", w32)
    _check(res, "k_kv4_join", 8)


@needs_hipcc
def test_cache_and_verification_kernels_keep_their_waves(tmp_path):
    res = _resources("kv4.hip", tmp_path)
    _check(res, "k_kv4_append", 8)
    _check(res, "k_kv4_read", 8)
    res = _resources("verify.hip", tmp_path)
    _check(res, "k_verify_scan", 8)
    _check(res, "k_verify_draw", 5)
