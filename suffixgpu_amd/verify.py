"""verify_draft: which drafted tokens the target model keeps, and the next one.

The step after the drafter's: the target has run over the drafted tokens and
its logits say, position by position, whether the draft stays.  The result is
``propose_with_update``'s ``sampled_token_ids``, so the loop closes on the
device without a host read.  No counterpart in the reference, whose verifier is
the engine's (its tests mimic one, suffix_gpu tests/test_verification.py).
"""

from __future__ import annotations

import torch

from suffixgpu_amd import _lib
from suffixgpu_amd._lib import check, lib, ptr, require_gpu, stream_of


# (device, stream) -> (counters, scratch).  The counters are zero between calls
# (every call leaves them so), the scratch is anything; two calls that share
# them are ordered by their stream.  Calls recorded into a HIP graph share a
# pair of their own per device (replays must not overlap each other): eager
# calls see to its size, so that a capture after a first eager call of that size
# records no fill.  Outgrown pairs of graphs are kept, a graph may hold them.
_workspaces: dict[tuple, tuple[torch.Tensor, torch.Tensor]] = {}
_outgrown: list[tuple[torch.Tensor, torch.Tensor]] = []


def _workspace(dev: torch.device, stream: int, nc: int, ns: int):
    capturing = torch.cuda.is_current_stream_capturing()
    for key in (((dev, "graph"),) if capturing
                else ((dev, "graph"), (dev, stream))):
        ws = _workspaces.get(key)
        if ws is None or ws[0].numel() < nc or ws[1].numel() < ns:
            if ws is not None:
                if key[1] == "graph":
                    _outgrown.append(ws)
                nc2 = max(nc, 2 * ws[0].numel())
                ns2 = max(ns, 2 * ws[1].numel())
            else:
                nc2, ns2 = max(nc, 1 << 16), max(ns, 1 << 18)
            ws = (torch.zeros(nc2, dtype=torch.uint8, device=dev),
                  torch.empty(ns2, dtype=torch.uint8, device=dev))
            _workspaces[key] = ws
    return ws


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
    drafts.

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
    stream.
    """
    require_gpu(logits, draft, num_valid, uniform, noise, temperature,
                draft_probs)
    if logits.dim() != 3 or logits.shape[1] < 1 or logits.shape[2] < 1:
        raise ValueError("logits must be [B, K + 1, V]")
    code = _lib.DTYPE_CODES.get(logits.dtype)
    if code is None:
        raise ValueError("logits must be bfloat16, float16 or float32")
    if logits.stride(2) != 1 and logits.shape[2] > 1:
        raise ValueError("logits must be contiguous along the vocabulary")
    b, k1, v = logits.shape
    dev = logits.device
    dense = [("draft", draft, (b, k1 - 1), torch.int32),
             ("num_valid", num_valid, (b,), torch.int32)]
    if not greedy:
        if uniform is None or noise is None:
            raise ValueError("uniform and noise are needed unless greedy")
        dense += [("uniform", uniform, (b, k1 - 1), torch.float32),
                  ("noise", noise, (b, v), torch.float32)]
        if temperature is not None:
            dense.append(("temperature", temperature, (b,), torch.float32))
        if draft_probs is not None:
            dense.append(("draft_probs", draft_probs, (b, k1 - 1, v),
                          torch.float32))
    for name, t, shape, dt in dense:
        if t.dtype != dt or t.device != dev or t.shape != shape:
            raise ValueError(f"{name} must be a {dt} tensor of shape "
                             f"{list(shape)} on {dev}")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    sampled = torch.empty(b, k1, dtype=torch.int32, device=dev)
    count = torch.empty(b, dtype=torch.int32, device=dev)
    if b == 0:
        return sampled, count
    L = lib()
    stream = stream_of(dev)
    counters, scratch = _workspace(dev, stream,
                                   L.sfx_verify_counter_bytes(b, k1 - 1, v),
                                   L.sfx_verify_workspace_size(b, k1 - 1, v))
    args = _lib.SfxVerify(
        logits.data_ptr(), code, int(greedy), b, k1 - 1, v,
        logits.stride(0), logits.stride(1), draft.data_ptr(),
        num_valid.data_ptr(),
        None if greedy else uniform.data_ptr(),
        None if greedy else noise.data_ptr(),
        None if greedy else ptr(temperature),
        None if greedy else ptr(draft_probs),
        sampled.data_ptr(), count.data_ptr())
    check(L.sfx_verify_draft(args, counters.data_ptr(), counters.numel(),
                             scratch.data_ptr(), scratch.numel(), stream),
          "verify_draft")
    return sampled, count
