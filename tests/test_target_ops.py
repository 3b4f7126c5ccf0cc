"""The target-side operators without a GPU: host checks of their C entry points
and of their Python forms, and the oracle's own ground."""

from __future__ import annotations

import ctypes
import importlib
import threading
import time

import numpy as np
import pytest
import torch

from oracle import target
from suffixgpu_amd import KV4Cache, _lib, verify_draft
from suffixgpu_amd.kv4 import block_bytes

# the module; the package's name of it is the function
verify = importlib.import_module("suffixgpu_amd.verify")


def cache(**kw):
    c = dict(pages=0x100000, num_pages=4, heads=2, head_dim=128, page_size=64,
             dtype=0, table=0x200000, table_width=2, table_stride=2)
    c.update(kw)
    return _lib.SfxKv4(**c)


HEADS = _lib.SfxHeads(0x300000, 256, 256, 128)


def test_block_bytes():
    lib = _lib.lib()
    for d in (64, 128, 256):
        assert lib.sfx_kv4_block_bytes(d) == block_bytes(d)
        assert block_bytes(d) % 16 == 0
    assert lib.sfx_kv4_block_bytes(96) == 0


@pytest.mark.parametrize("bad", [
    dict(head_dim=96), dict(page_size=48), dict(page_size=16),
    dict(page_size=1 << 17), dict(heads=0), dict(dtype=2), dict(dtype=-1),
    dict(num_pages=-1), dict(pages=None), dict(pages=0x100008),
    dict(table=None), dict(table_width=-1), dict(table_width=1 << 25)])
def test_cache_geometry_is_checked_on_the_host(bad):
    lib = _lib.lib()
    c = cache(**bad)
    assert lib.sfx_kv4_append(c, HEADS, HEADS, 0, 1, None, 0, None, 0,
                              None) == -1
    assert lib.sfx_kv4_read(c, 0, 1, None, 0, None, 0, None, None, None) == -1
    assert lib.sfx_kv4_attend(c, HEADS, 0, 1, 4, None, 0, None, 0, 1.0, None,
                              None, 0, None) == -1
    assert lib.sfx_kv4_attend_workspace_size(c, 1, 1, 4) == 0


def test_cache_calls_are_checked_on_the_host():
    lib = _lib.lib()
    c = cache()
    # an empty batch is no error and launches nothing
    assert lib.sfx_kv4_append(c, HEADS, HEADS, 0, 1, None, 0, None, 0,
                              None) == 0
    assert lib.sfx_kv4_attend(c, HEADS, 0, 1, 4, None, 0, None, 0, 1.0, None,
                              None, 0, None) == 0
    for b, t in ((-1, 1), (1, -1), (65536, 1), (1, 1 << 40)):
        assert lib.sfx_kv4_append(c, HEADS, HEADS, b, t, 0x1000, 0, None, 0,
                                  None) == -1
        assert lib.sfx_kv4_attend(c, HEADS, b, t, 4, 0x1000, 0, None, 0, 1.0,
                                  0x2000, 0x3000, 1 << 40, None) == -1
    none = _lib.SfxHeads(None, 0, 0, 0)
    assert lib.sfx_kv4_append(c, none, HEADS, 1, 1, 0x1000, 0, None, 0,
                              None) == -1
    assert lib.sfx_kv4_append(c, HEADS, HEADS, 1, 1, None, 0, None, 0,
                              None) == -1
    assert lib.sfx_kv4_read(c, 1, 1, 0x1000, 0, None, 0, 0x2008, 0x3000,
                            None) == -1
    # query heads that do not divide, a missing length, a short workspace
    assert lib.sfx_kv4_attend(c, HEADS, 1, 1, 3, 0x1000, 0, None, 0, 1.0,
                              0x2000, 0x3000, 1 << 40, None) == -1
    assert lib.sfx_kv4_attend(c, HEADS, 1, 1, 4, None, 0, None, 0, 1.0,
                              0x2000, 0x3000, 1 << 40, None) == -1
    big = cache(table_width=4096, num_pages=1 << 20)
    need = lib.sfx_kv4_attend_workspace_size(big, 1, 1, 4)
    assert need > 0
    assert lib.sfx_kv4_attend(big, HEADS, 1, 1, 4, 0x1000, 0, None, 0, 1.0,
                              0x2000, 0x3000, need - 1, None) == -1


def test_verify_is_checked_on_the_host():
    lib = _lib.lib()

    def args(**kw):
        a = dict(logits=0x100000, dtype=0, all_greedy=0, batch=2, k=3,
                 vocab=100, stride_b=400, stride_j=100, draft=0x1000,
                 num_valid=0x2000, uniform=0x3000, noise=0x4000,
                 temperature=None, draft_probs=None, sampled=0x5000,
                 count=0x6000)
        a.update(kw)
        return _lib.SfxVerify(**a)

    need = lib.sfx_verify_workspace_size(2, 3, 100)
    assert need > 0
    for bad in (dict(dtype=3), dict(batch=-1), dict(k=-1), dict(k=5000),
                dict(vocab=0), dict(vocab=1 << 30), dict(logits=None),
                dict(draft=None), dict(num_valid=None), dict(uniform=None),
                dict(noise=None), dict(sampled=None), dict(count=None),
                dict(batch=1 << 24)):
        assert lib.sfx_verify_draft(args(**bad), 0x7000, 1 << 30, 0x8000,
                                    1 << 30, None) == -1
    zeros = lib.sfx_verify_counter_bytes(2, 3, 100)
    assert zeros > 0
    for c, nc, w, nw in ((0x7000, zeros, 0x8000, need - 1),
                         (0x7000, zeros - 1, 0x8000, need),
                         (0x7008, zeros, 0x8000, need),
                         (0x7000, zeros, 0x8008, need),
                         (None, zeros, 0x8000, need),
                         (0x7000, zeros, None, need)):
        assert lib.sfx_verify_draft(args(), c, nc, w, nw, None) == -1
    assert lib.sfx_verify_draft(args(batch=0), None, 0, None, 0, None) == 0
    assert lib.sfx_verify_workspace_size(0, 3, 100) == 0


def test_no_cpu_path():
    with pytest.raises(_lib.SuffixGPUError):
        KV4Cache(4, 2, 64, device="cpu")
    x = torch.zeros(1, 2, 8)
    with pytest.raises(_lib.SuffixGPUError):
        verify_draft(x, torch.zeros(1, 1, dtype=torch.int32),
                     torch.zeros(1, dtype=torch.int32), greedy=True)


def test_struct_sizes():
    assert ctypes.sizeof(_lib.SfxKv4) == 72
    assert ctypes.sizeof(_lib.SfxHeads) == 32
    assert ctypes.sizeof(_lib.SfxVerify) == 120


# ------------------------------------------------------------- the oracle
def test_oracle_rounding_by_distance():
    """round_e2m1 takes the nearest level, the even one of two."""
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.uniform(0, 8, 4000), np.arange(0, 8, 0.125)])
    got = target.round_e2m1(x, np.float64(1.0))
    dist = np.abs(x[:, None] - target.LEVELS)
    best = dist.min(axis=1)
    assert (np.abs(got - x) == best).all()
    two = (dist == best[:, None]).sum(axis=1) == 2
    assert two.sum() >= 7
    assert (np.searchsorted(target.LEVELS, got[two]) % 2 == 0).all()


def test_oracle_key_scales():
    a = np.zeros((4, 32))
    a[:, 0] = [7.0, 7.5, 3.5, 6.0]
    q = target.quantize_k(a, False)
    # 7 rounds to 6 at 2^0, 7.5 to 4 at 2^1, 3.5 is 7 at 2^-1
    np.testing.assert_array_equal(q[:, 0], [6.0, 8.0, 3.0, 6.0])


def test_oracle_verify_by_hand():
    x = np.log(np.array([[[0.5, 0.3, 0.2], [0.1, 0.1, 0.8]]]))
    d, n = np.array([[1]]), np.array([1])
    e = np.ones((1, 3))
    # 0.29 < 0.3 keeps the draft, the token after it is the likeliest
    s, c, _ = target.verify(x, d, n, np.array([[0.29]]), e, None)
    assert s.tolist() == [[1, 2]] and c.tolist() == [2]
    # rejected: drawn from the others
    s, c, _ = target.verify(x, d, n, np.array([[0.31]]), e, None)
    assert s.tolist() == [[0, -1]] and c.tolist() == [1]
    # with draft probabilities: 0.5 * 0.9 >= 0.3, and r = (0.45, 0, 0.15)
    q = np.array([[[0.05, 0.9, 0.05]]])
    e = np.array([[4.0, 1.0, 1.0]])
    s, c, _ = target.verify(x, d, n, np.array([[0.5]]), e, None, q)
    assert s.tolist() == [[2, -1]]


def test_oracle_attention_by_hand():
    k = np.zeros((1, 2, 1, 32))
    v = np.zeros((1, 2, 1, 32))
    v[0, 0, 0, 0], v[0, 1, 0, 0] = 1.0, 3.0
    q = np.zeros((1, 2, 1, 32))
    out, _ = target.attend(q, k, v, np.ones((1, 2, 1, 1)), [2], [2])
    assert out[0, :, 0, 0].tolist() == [1.0, 2.0]


class _FakeLib:
    """sfx_verify_draft that takes a while, as two launches do, and says whether
    another call came in between."""

    def __init__(self):
        self.inside = self.most = 0
        self.lock = threading.Lock()

    def sfx_verify_counter_bytes(self, *_):
        return 64

    def sfx_verify_workspace_size(self, *_):
        return 64

    def sfx_verify_draft(self, *_):
        with self.lock:
            self.inside += 1
            self.most = max(self.most, self.inside)
        time.sleep(0.02)
        with self.lock:
            self.inside -= 1
        return 0


def test_verify_calls_of_two_threads_do_not_interleave(monkeypatch):
    """A call's two launches hand their counters over, which calls on one stream
    share: no other thread's launch comes between them."""
    fake = _FakeLib()
    monkeypatch.setattr(verify, "lib", lambda: fake)
    monkeypatch.setattr(verify, "require_gpu", lambda *_: None)
    monkeypatch.setattr(verify, "stream_of", lambda _: 0)
    monkeypatch.setattr(verify, "_workspaces", {})
    monkeypatch.setattr(verify, "_sizes", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing",
                        lambda: False)
    x = torch.zeros(1, 2, 8)
    draft, num = (torch.zeros(1, 1, dtype=torch.int32),
                  torch.zeros(1, dtype=torch.int32))
    errors = []

    def work():
        try:
            for _ in range(3):
                verify_draft(x, draft, num, greedy=True)
        except Exception as e:          # a thread's own exception is lost
            errors.append(e)

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and fake.most == 1


def test_verify_counters_of_a_failed_call_are_not_used_again(monkeypatch):
    """A call that fails between its launches leaves its counters anyhow: the next
    one gets others, which are zero."""
    seen = []

    class Fake(_FakeLib):
        def sfx_verify_draft(self, _, counters, nbytes, *__):
            words = (ctypes.c_uint8 * nbytes).from_address(counters)
            seen.append(bytes(words) == bytes(nbytes))
            words[0] = 1
            return 1 if len(seen) == 1 else 0

    fake = Fake()
    monkeypatch.setattr(verify, "lib", lambda: fake)
    monkeypatch.setattr(verify, "require_gpu", lambda *_: None)
    monkeypatch.setattr(verify, "stream_of", lambda _: 0)
    monkeypatch.setattr(verify, "_workspaces", {})
    monkeypatch.setattr(verify, "_sizes", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing",
                        lambda: False)
    x = torch.zeros(1, 2, 8)
    draft, num = (torch.zeros(1, 1, dtype=torch.int32),
                  torch.zeros(1, dtype=torch.int32))
    with pytest.raises(_lib.SuffixGPUError):
        verify_draft(x, draft, num, greedy=True)
    verify_draft(x, draft, num, greedy=True)
    assert seen == [True, True]
