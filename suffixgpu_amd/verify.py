"""verify_draft: which drafted tokens the target model keeps, and the next one.

The step after the drafter's: the target has run over the drafted tokens and
its logits say, position by position, whether the draft stays.  The result is
``propose_with_update``'s ``sampled_token_ids``, so the loop closes on the
device without a host read.  No counterpart in the reference, whose verifier is
the engine's (its tests mimic one, suffix_gpu tests/test_verification.py).
"""

from __future__ import annotations

import threading

import torch

from suffixgpu_amd import _lib
from suffixgpu_amd._lib import (check, elsewhere, lib, require_gpu,
                                stream_of)


# Counters and scratch, as (counters, scratch, counters' address, bytes, scratch's
# address, bytes), by device and stream.  The counters are zero between calls
# (every call leaves them so), the scratch is anything.  Calls that share them are
# ordered by their stream, each call's two launches side by side: the C call lets
# other threads run, so it is made with `_enqueue` held.  A call recorded into a HIP graph has a pair out of
# the graph's own memory, cleared by a node of the graph: graphs recorded on one
# stream may be replayed on others, at the same time and in any order.
_workspaces: dict[tuple, tuple] = {}
_enqueue = threading.Lock()


def _new_workspace(dev: torch.device, nc: int, ns: int) -> tuple:
    c = torch.zeros(nc, dtype=torch.uint8, device=dev)
    s = torch.empty(ns, dtype=torch.uint8, device=dev)
    return c, s, c.data_ptr(), nc, s.data_ptr(), ns


def _workspace(dev: torch.device, stream: int, nc: int, ns: int) -> tuple:
    """The pair for `stream`, with at least nc and ns bytes."""
    if torch.cuda.is_current_stream_capturing():
        return _new_workspace(dev, nc, ns)
    ws = _workspaces.get((dev, stream))
    if ws is None or ws[3] < nc or ws[5] < ns:
        ws = _workspaces[dev, stream] = _new_workspace(
            dev, max(2 * nc, 1 << 16), max(2 * ns, 1 << 18))
    return ws


# Workspace bytes by (batch, drafts, vocabulary).
_sizes: dict[tuple, tuple[int, int]] = {}


def _need(name: str, t: torch.Tensor, shape: tuple, dtype: torch.dtype,
          dev: torch.device) -> int:
    if (t.dtype is not dtype or t.device != dev or t.shape != shape
            or not t.is_contiguous()):
        require_gpu(t)
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape "
                         f"{list(shape)} on {dev}")
    return t.data_ptr()


def verify_draft(logits: torch.Tensor, draft: torch.Tensor,
                 num_valid: torch.Tensor,
                 uniform: torch.Tensor | None = None,
                 noise: torch.Tensor | None = None,
                 temperature: torch.Tensor | None = None,
                 draft_probs: torch.Tensor | None = None,
                 greedy: bool = False):
    """Verify ``draft`` [B, K] (int32, ``num_valid`` [B] of each row) against
    ``logits`` [B, K + 1, V] (bfloat16, float16 or float32; any strides but a
    contiguous vocabulary), position j holding the target's logits after j
    drafts.  An id outside the vocabulary ends a row's drafts as num_valid does.

    With p = softmax(logits / temperature), draft j stays iff
    ``uniform[b, j] * q < p[draft]``; q is ``draft_probs[b, j, draft]``
    ([B, K, V] float32), or 1 for a drafter that gives none, as this package's.
    After the kept ones a token is drawn: from max(p - q, 0) at the first draft
    that does not stay, from p when all do -- the token with the largest
    probability / ``noise[b, token]``, the lowest on ties.  ``uniform`` [B, K]
    lies in [0, 1), ``noise`` [B, V] is exponentially distributed
    (``torch.empty(B, V, device=...).exponential_()``), both float32.

    ``temperature`` [B] float32 (default 1); rows at 0 are greedy: a draft
    stays iff it is the first largest logit, which is also the token drawn.
    ``greedy=True`` says so of every row, and needs neither random numbers nor
    temperatures.  NaN logits count as -inf.  A position without any logit
    above -inf keeps and draws nothing.

    Returns (sampled [B, K + 1] int32: kept drafts, the drawn token, then -1;
    count [B] int32).  No host synchronisation; two launches on the current
    stream, and a fill before them where they are recorded into a HIP graph.
    """
    require_gpu(logits)
    dev = logits.device
    if elsewhere(dev):
        with torch.cuda.device(dev):
            return verify_draft(logits, draft, num_valid, uniform, noise,
                                temperature, draft_probs, greedy)
    if logits.dim() != 3:
        raise ValueError("logits must be [B, K + 1, V]")
    b, k1, v = logits.shape
    if k1 < 1 or v < 1:
        raise ValueError("logits must be [B, K + 1, V]")
    code = _lib.DTYPE_CODES.get(logits.dtype)
    if code is None:
        raise ValueError("logits must be bfloat16, float16 or float32")
    sb, sj, sv = logits.stride()
    if sv != 1 and v > 1:
        raise ValueError("logits must be contiguous along the vocabulary")
    k = k1 - 1
    dp = _need("draft", draft, (b, k), torch.int32, dev)
    np_ = _need("num_valid", num_valid, (b,), torch.int32, dev)
    up = ep = tp = qp = None
    if not greedy:
        if uniform is None or noise is None:
            raise ValueError("uniform and noise are needed unless greedy")
        up = _need("uniform", uniform, (b, k), torch.float32, dev)
        ep = _need("noise", noise, (b, v), torch.float32, dev)
        if temperature is not None:
            tp = _need("temperature", temperature, (b,), torch.float32, dev)
        if draft_probs is not None:
            qp = _need("draft_probs", draft_probs, (b, k, v), torch.float32,
                       dev)
    sampled = torch.empty(b, k1, dtype=torch.int32, device=dev)
    count = torch.empty(b, dtype=torch.int32, device=dev)
    if b == 0:
        return sampled, count
    L = lib()
    size = _sizes.get((b, k, v))
    if size is None:
        size = _sizes[b, k, v] = (L.sfx_verify_counter_bytes(b, k, v),
                                  L.sfx_verify_workspace_size(b, k, v))
    stream = stream_of(dev)
    args = _lib.SfxVerify(logits.data_ptr(), code, int(greedy), b, k, v, sb,
                          sj, dp, np_, up, ep, tp, qp, sampled.data_ptr(),
                          count.data_ptr())
    with _enqueue:
        ws = _workspace(dev, stream, *size)
        rc = L.sfx_verify_draft(args, *ws[2:], stream)
        if rc:      # its counters may be anything
            _workspaces.pop((dev, stream), None)
    check(rc, "verify_draft")
    return sampled, count
