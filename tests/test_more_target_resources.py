"""Registers and scratch of the kernels of token_logprobs, PagePool and attention
over selected blocks, from the compiler's resource report: as those that they stand
beside, they are laid out for so many waves on a SIMD, and what goes to scratch
memory says no word."""

from __future__ import annotations

from tests.test_kernel_resources import _resources
from tests.test_target_resources import _check, needs_hipcc


@needs_hipcc
def test_logprob_and_page_kernels_keep_their_waves(tmp_path):
    res = _resources("logprobs.hip", tmp_path)
    _check(res, "k_logprobs_scan", 7)
    _check(res, "k_logprobs_join", 8)
    res = _resources("pages.hip", tmp_path)
    # (1,024 threads: four waves a SIMD)
    _check(res, "k_pages_resize", 4)
    _check(res, "k_pages_plan", 4)
    _check(res, "k_pages_move", 8)
    _check(res, "k_pages_slots", 8)


@needs_hipcc
def test_block_kernels_keep_their_waves(tmp_path):
    res = _resources("kv4_select.hip", tmp_path)
    _check(res, "k_kv4_bounds", 7)
    # by head size, which the mangled name has as the first argument
    for d, waves in ((64, 7), (128, 7), (256, 4)):
        for half in (0, 1):
            _check(res, f"k_kv4_selectILi{d}ELb{half}ELb0E", waves)
            # (few tokens: two workgroups of eight waves a CU)
            _check(res, f"k_kv4_selectILi{d}ELb{half}ELb1E", 4)
        _check(res, f"k_kv4_scoresILi{d}E", waves)
    _check(res, "k_kv4_pick_wide", 7)
    _check(res, "k_kv4_pick_far", 8)
    res = _resources("kv4_blocks.hip", tmp_path)
    for d, waves in ((64, 4), (128, 4), (256, 2)):
        _check(res, f"k_kv4_attend_blocksILi{d}E", waves)
    _check(res, "k_kv4_union", 8)
    _check(res, "k_kv4_join_blocks", 8)
