"""token_logprobs, PagePool and attention over selected blocks without a GPU: host
checks of their C entry points, their refusals, and the oracle's own ground."""

from __future__ import annotations

import ctypes
import shutil
import subprocess
import threading
import time

import numpy as np
import pytest
import torch

from oracle import target
from suffixgpu_amd import KV4Cache, PagePool, _lib, pages, token_logprobs
from tests.test_abi import ROCM_INCLUDE, ROOT
from tests.test_target_ops import HEADS, cache

BOUNDS = _lib.SfxKv4Bounds(0x400000, 0x500000)


# ------------------------------------------------------- log probabilities
def logprob_args(**kw):
    a = dict(logits=0x100000, dtype=0, batch=2, positions=3, vocab=100,
             stride_b=300, stride_j=100, tokens=0x1000, temperature=None,
             top=4, logprob=0x2000, entropy=0x3000, top_tokens=0x4000,
             top_logprobs=0x5000)
    a.update(kw)
    return _lib.SfxLogprobs(**a)


def test_logprobs_are_checked_on_the_host():
    lib = _lib.lib()
    need = lib.sfx_logprobs_workspace_size(2, 3, 100, 4)
    assert need > 0
    for bad in (dict(dtype=3), dict(dtype=-1), dict(batch=-1),
                dict(positions=-1), dict(vocab=0), dict(vocab=1 << 30),
                dict(top=-1), dict(top=_lib.LOGPROBS_TOP + 1),
                dict(logits=None), dict(tokens=None), dict(logprob=None),
                dict(entropy=None), dict(top_tokens=None),
                dict(top_logprobs=None), dict(batch=1 << 24),
                dict(batch=1 << 20, positions=1 << 20)):
        assert lib.sfx_token_logprobs(logprob_args(**bad), 0x8000, 1 << 40,
                                      None) == -1
    for w, n in ((0x8000, need - 1), (0x8008, need), (None, need)):
        assert lib.sfx_token_logprobs(logprob_args(), w, n, None) == -1
    assert lib.sfx_token_logprobs(None, 0x8000, need, None) == -1
    for empty in (dict(batch=0), dict(positions=0)):
        assert lib.sfx_token_logprobs(logprob_args(**empty), None, 0,
                                      None) == 0
    assert lib.sfx_logprobs_workspace_size(0, 3, 100, 4) == 0
    assert lib.sfx_logprobs_workspace_size(2, 3, 100, 33) == 0


# ------------------------------------------------------------- page tables
def pool(**kw):
    p = dict(free_pages=0x1000, num_free=0x2000, held=0x3000, table=0x4000,
             num_pages=10, rows=4, table_width=5, page_size=64, plan=0x5000)
    p.update(kw)
    return _lib.SfxPages(**p)


def test_pages_are_checked_on_the_host():
    lib = _lib.lib()
    for bad in (dict(free_pages=None), dict(num_free=None), dict(held=None),
                dict(table=None), dict(plan=None), dict(num_pages=-1),
                dict(num_pages=1 << 31), dict(rows=0),
                dict(rows=_lib.PAGES_ROWS + 1), dict(table_width=0),
                dict(table_width=1 << 25), dict(page_size=0),
                dict(page_size=48), dict(page_size=1 << 17)):
        assert lib.sfx_pages_resize(pool(**bad), 0x6000, 0, 1, 0x7000,
                                    None) == -1
        assert lib.sfx_pages_slots(pool(**bad), 0x6000, 0, None, 0, 1, 1,
                                   0x7000, None) == -1
    p = pool()
    for n in (-1, 5):
        assert lib.sfx_pages_resize(p, 0x6000, 0, n, 0x7000, None) == -1
        assert lib.sfx_pages_slots(p, 0x6000, 0, None, 0, n, 1, 0x7000,
                                   None) == -1
    assert lib.sfx_pages_resize(p, None, 0, 1, 0x7000, None) == -1
    assert lib.sfx_pages_resize(p, 0x6000, 0, 1, None, None) == -1
    assert lib.sfx_pages_slots(p, None, 0, None, 0, 1, 1, 0x7000, None) == -1
    assert lib.sfx_pages_slots(p, 0x6000, 0, None, 0, 1, 1, None, None) == -1
    assert lib.sfx_pages_slots(p, 0x6000, 0, None, 0, 1, -1, 0x7000,
                               None) == -1
    assert lib.sfx_pages_resize(None, 0x6000, 0, 1, 0x7000, None) == -1
    # nothing to do is no error and launches nothing
    assert lib.sfx_pages_resize(p, None, 0, 0, None, None) == 0
    assert lib.sfx_pages_slots(p, None, 0, None, 0, 0, 4, None, None) == 0
    assert lib.sfx_pages_slots(p, None, 0, None, 0, 2, 0, None, None) == 0


def test_resizes_of_two_threads_do_not_interleave(monkeypatch):
    """A call's two launches hand a plan over, which the pool has one of."""
    class Fake:
        inside = most = 0
        lock = threading.Lock()

        def sfx_pages_resize(self, *_):
            with self.lock:
                self.inside += 1
                self.most = max(self.most, self.inside)
            time.sleep(0.02)
            with self.lock:
                self.inside -= 1
            return 0

    fake = Fake()
    monkeypatch.setattr(pages, "lib", lambda: fake)
    monkeypatch.setattr(pages, "stream_of", lambda _: 0)
    p = object.__new__(PagePool)
    p.device, p.rows, p._view = torch.device("cpu"), 2, None
    p._enqueue = threading.Lock()
    lens = torch.zeros(2, dtype=torch.int32)
    threads = [threading.Thread(target=p.resize, args=(lens,))
               for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert fake.most == 1


# --------------------------------------------------------- selected blocks
@pytest.mark.parametrize("bad", [
    dict(head_dim=96), dict(page_size=48), dict(heads=0), dict(dtype=2),
    dict(num_pages=-1), dict(pages=None), dict(table=None),
    dict(table_width=1 << 25)])
def test_cache_geometry_is_checked(bad):
    lib = _lib.lib()
    c = cache(**bad)
    assert lib.sfx_kv4_bounds_update(c, BOUNDS, 0, 1, None, 0, None, 0,
                                     None) == -1
    assert lib.sfx_kv4_select(c, BOUNDS, HEADS, 0, 1, 4, None, 0, None, 0, 4, 1,
                              1, None, None, 0, None) == -1
    assert lib.sfx_kv4_attend_blocks(c, HEADS, 0, 1, 4, None, 4, None, 0, None,
                                     0, 1.0, None, None, 0, None) == -1
    assert lib.sfx_kv4_select_workspace_size(c, 1, 1) == 0
    assert lib.sfx_kv4_attend_blocks_workspace_size(c, 1, 2, 4, 4) == 0


def test_selection_is_checked_on_the_host():
    lib = _lib.lib()
    c = cache()

    def select(c=c, bounds=BOUNDS, q=HEADS, b=1, t=1, hq=4, kv=0x1000, n=4,
               first=1, recent=1, out=0x2000, ws=None, nws=0):
        return lib.sfx_kv4_select(c, bounds, q, b, t, hq, kv, 0, None, 0, n,
                                  first, recent, out, ws, nws, None)

    for bad in (dict(bounds=None), dict(q=None), dict(b=-1), dict(b=65536),
                dict(t=-1), dict(t=1 << 25), dict(b=65535, t=1 << 10),
                dict(hq=0), dict(hq=3), dict(kv=None), dict(n=1),
                dict(n=32769), dict(first=-1), dict(first=4), dict(recent=0),
                dict(recent=4), dict(out=None), dict(out=None),
                dict(q=_lib.SfxHeads(None, 0, 0, 0)),
                dict(bounds=_lib.SfxKv4Bounds(None, 0x1000)),
                dict(bounds=_lib.SfxKv4Bounds(0x1008, 0x1000)),
                dict(bounds=_lib.SfxKv4Bounds(0x1000, None))):
        assert select(**bad) == -1, bad
    assert select(b=0) == 0 and select(t=0) == 0
    # a workspace where a workgroup does not hold a row's keys
    assert lib.sfx_kv4_select_workspace_size(c, 1, 1) == 0
    wide = cache(table_width=1024)
    need = lib.sfx_kv4_select_workspace_size(wide, 2, 3)
    assert need == 2 * 3 * 2 * 2048 * 4
    for ws, n in ((None, need), (0x3000, need - 1), (0x3008, need)):
        assert select(c=wide, b=2, t=3, ws=ws, nws=n) == -1
    for bad in (dict(batch=-1), dict(batch=65536), dict(tokens=-1),
                dict(tokens=1 << 40), dict(start=None)):
        a = dict(batch=1, tokens=1, start=0x1000)
        a.update(bad)
        assert lib.sfx_kv4_bounds_update(c, BOUNDS, a["batch"], a["tokens"],
                                         a["start"], 0, None, 0, None) == -1
    assert lib.sfx_kv4_bounds_update(c, None, 1, 1, 0x1000, 0, None, 0,
                                     None) == -1


def test_attention_over_blocks_is_checked_on_the_host():
    lib = _lib.lib()
    c = cache()

    def attend(q=HEADS, b=1, t=1, hq=4, sel=0x1000, n=40, kv=0x2000,
               out=0x3000, ws=0x4000, nws=1 << 40):
        return lib.sfx_kv4_attend_blocks(c, q, b, t, hq, sel, n, kv, 0, None, 0,
                                         1.0, out, ws, nws, None)

    for bad in (dict(q=None), dict(q=_lib.SfxHeads(None, 0, 0, 0)), dict(b=-1),
                dict(b=65536), dict(t=-1), dict(t=1 << 40), dict(hq=0),
                dict(hq=3), dict(sel=None), dict(n=0), dict(n=32769),
                dict(kv=None), dict(out=None), dict(out=0x3008), dict(ws=None),
                dict(ws=0x4008), dict(nws=0)):
        assert attend(**bad) == -1, bad
    assert attend(b=0) == 0 and attend(t=0) == 0
    # a list of 40 for each of two KV heads is split, one of 8 is not
    assert lib.sfx_kv4_attend_blocks_workspace_size(c, 1, 1, 4, 40) > 0
    assert lib.sfx_kv4_attend_blocks_workspace_size(c, 1, 1, 4, 8) == 0


def test_no_cpu_path():
    with pytest.raises(_lib.SuffixGPUError):
        PagePool(4, 2, 2, device="cpu")
    with pytest.raises(_lib.SuffixGPUError):
        KV4Cache(4, 2, 64, device="cpu", bounds=True)
    with pytest.raises(_lib.SuffixGPUError):
        token_logprobs(torch.zeros(1, 2, 8), torch.zeros(1, 2,
                                                         dtype=torch.int32))


PROBE = r"""
#include <stddef.h>
#include <stdio.h>
#include "suffixgpu_amd.h"
#define F(T, f) printf(#T "." #f " %zu\n", offsetof(T, f))
#define S(T) printf(#T " %zu\n", sizeof(T))
int main(void) {
  S(sfx_logprobs); F(sfx_logprobs, dtype); F(sfx_logprobs, stride_j);
  F(sfx_logprobs, temperature); F(sfx_logprobs, top);
  F(sfx_logprobs, top_logprobs);
  S(sfx_pages); F(sfx_pages, table); F(sfx_pages, page_size);
  F(sfx_pages, plan);
  S(sfx_kv4_bounds); F(sfx_kv4_bounds, unit);
  printf("TOP %d\nROWS %d\n", SFX_LOGPROBS_TOP, SFX_PAGES_ROWS);
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("gcc") is None
                    or not (ROCM_INCLUDE / "hip").is_dir(),
                    reason="needs gcc and the ROCm headers")
def test_structs_are_the_headers(tmp_path):
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text(PROBE)
    subprocess.run(["gcc", "-D__HIP_PLATFORM_AMD__", f"-I{ROOT / 'include'}",
                    f"-I{ROCM_INCLUDE}", str(src), "-o", str(exe)],
                   check=True, capture_output=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True,
                         text=True).stdout
    c = dict(line.rsplit(" ", 1) for line in out.strip().splitlines())
    assert int(c.pop("TOP")) == _lib.LOGPROBS_TOP
    assert int(c.pop("ROWS")) == _lib.PAGES_ROWS
    mirrors = {"sfx_logprobs": _lib.SfxLogprobs, "sfx_pages": _lib.SfxPages,
               "sfx_kv4_bounds": _lib.SfxKv4Bounds}
    for key, val in c.items():
        t, _, f = key.partition(".")
        got = (getattr(mirrors[t], f).offset if f
               else ctypes.sizeof(mirrors[t]))
        assert got == int(val), key


# --------------------------------------------------------------- the oracle
def test_oracle_bounds_hold_the_keys():
    rng = np.random.default_rng(1)
    for scale in (1e-40, 1e-3, 1.0, 1e30):
        k = target.quantize_k(rng.standard_normal((32, 64)) * scale, False)
        lo, hi, u = target.key_bounds(k)
        assert (lo * 2.0 ** u <= k.min(axis=0)).all()
        assert (hi * 2.0 ** u >= k.max(axis=0)).all()
        # within a unit of the least and the largest, 64 units at most the
        # largest magnitude
        if u > -100:
            assert 64 <= np.abs(k).max() / 2.0 ** u < 128
            assert (hi * 2.0 ** u - k.max(axis=0) < 2.0 ** u).all()


def test_oracle_scores_bound_the_products():
    """P hi - N lo is at least the sum over the heads of q k, but for the query's
    rounding, for every key of a block."""
    rng = np.random.default_rng(2)
    q = rng.standard_normal((4, 64))
    k = target.quantize_k(rng.standard_normal((32, 64)), False)
    lo, hi, u = target.key_bounds(k)
    p, n = target.pack_query(q)
    assert max(p.max(), n.max()) in range(64, 128)
    pos, neg = np.maximum(q, 0).sum(axis=0), np.maximum(-q, 0).sum(axis=0)
    # what one of the 7-bit numbers' steps is worth
    step = max(pos.max(), neg.max()) / max(p.max(), n.max()) * (1 + 1 / 63)
    score = (p @ hi - n @ lo) * 2.0 ** u * step
    slack = step * (np.abs(hi) + np.abs(lo)).sum() * 2.0 ** u
    assert score + slack >= (q.sum(axis=0) @ k.T).max()


def test_oracle_selection_by_hand():
    # three blocks of one channel pair, largest keys 1, 3, 2 units
    def block(x):
        return [(np.array([0, 0]), np.array([x, 0]), 0)]
    b = [[block(1), block(3), block(2), block(0)]]
    q = np.zeros((1, 1, 1, 2))
    q[..., 0] = 1.0

    def got(n, first, recent, kv=128):
        return target.select_blocks(q, b, [kv], [1], 128, n, first,
                                    recent)[0, 0, 0].tolist()
    assert got(2, 0, 1) == [1, 3]
    assert got(3, 0, 1) == [1, 2, 3]
    assert got(3, 1, 1) == [0, 1, 3]
    assert got(3, 1, 2) == [0, 2, 3]
    assert got(2, 0, 1, kv=64) == [0, 1]
    assert got(2, 0, 1, kv=0) == [-1, -1]
    assert got(6, 1, 1) == [0, 1, 2, 3, -1, -1]


def test_oracle_attention_over_all_blocks_is_attention():
    rng = np.random.default_rng(3)
    k, v = rng.standard_normal((2, 1, 70, 1, 32))
    q = rng.standard_normal((1, 3, 2, 32))
    s = np.ones((1, 70, 1, 1))
    sel = np.array([[[[2, 0, 1, 0, -1, 7]]] * 3])
    one, b1 = target.attend(q, k, v, s, [70], [3])
    two, b2 = target.attend_blocks(q, sel, k, v, s, [70], [3])
    np.testing.assert_allclose(one, two, rtol=1e-12)
    np.testing.assert_allclose(b1, b2, rtol=1e-9)


def test_oracle_logprobs_by_hand():
    x = np.log(np.array([[[0.5, 0.25, 0.25], [0.1, 0.8, 0.1]]]))
    lp, h, ids, alt, _ = target.logprobs(x, np.array([[1, 3]]), None, 2)
    np.testing.assert_allclose(lp, [[np.log(0.25), 0.0]])
    np.testing.assert_allclose(h, [[1.5 * np.log(2), 0.0]])
    assert ids.tolist() == [[[0, 1], [-1, -1]]]
    np.testing.assert_allclose(alt[0, 0], np.log([0.5, 0.25]))
    lp, h, ids, alt, _ = target.logprobs(x, np.array([[1, 1]]), [0.0], 2)
    assert lp.tolist() == [[-np.inf, 0.0]] and h.tolist() == [[0.0, 0.0]]
    assert ids.tolist() == [[[0, 1], [1, 0]]]
    assert alt.tolist() == [[[0.0, -np.inf], [0.0, -np.inf]]]


def test_oracle_pages_by_hand():
    p = target.Pages(5, 3, 3, 10)
    assert p.resize([11, 5, 40]) == [20, 10, 20]     # two of the last three
    assert p.table().tolist() == [[0, 1, -1], [2, -1, -1], [3, 4, -1]]
    assert p.free == []
    # what comes back is free from the next call on
    assert p.resize([0, 25, -1]) == [0, 10, 20]
    assert p.free == [1, 0]
    assert p.resize([0, 25]) == [0, 30]
    assert p.table()[1].tolist() == [2, 0, 1]
    assert p.slots([0, 8], 4, [4, 3]).tolist() == [[-1] * 4, [28, 29, 0, -1]]
