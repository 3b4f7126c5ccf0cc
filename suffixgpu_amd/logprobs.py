"""token_logprobs: log probabilities of given tokens, with the entropy of their
distributions and the likeliest alternatives.

What a server reports beside the tokens that ``verify_draft`` gives, from the same
logits and temperatures.  No counterpart in the reference, whose sampling is the
engine's.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from suffixgpu_amd import _lib
from suffixgpu_amd._lib import (check, elsewhere, lib, require_gpu,
                                stream_of)


# Workspace bytes by (batch, positions, vocabulary, alternatives).
_sizes: dict[tuple, int] = {}


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor       # [B, J] float32
    entropy: torch.Tensor       # [B, J] float32
    top_tokens: torch.Tensor    # [B, J, top] int32
    top_logprobs: torch.Tensor  # [B, J, top] float32


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor,
                   temperature: torch.Tensor | None = None,
                   top: int = 0) -> TokenLogprobs:
    """Natural logarithms of p(token) for ``tokens`` [B, J] (int32) under
    p = softmax(``logits`` [B, J, V] / ``temperature`` [B]) (bfloat16, float16 or
    float32; any strides but a contiguous vocabulary), the entropy of p, and the
    ``top`` (up to 32) likeliest tokens with theirs, the lowest first on ties.

    p is ``verify_draft``'s: NaN logits count as -inf, a row at temperature 0 has
    all of p at the first largest logit.  ``verify_draft``'s ``sampled`` may be
    passed as it is: a position whose token is outside [0, V), as the -1 behind
    the drawn one, is not read and has (0, 0, -1, -inf).  Where fewer than ``top``
    logits are above -inf the rest of ``top_tokens`` is -1, of ``top_logprobs``
    -inf; without any, the log probability is -inf and the entropy 0.

    Serves a model; there are no gradients, and logits or temperatures that ask
    for them are refused.  No host synchronisation; two launches on the current
    stream, which may be recorded into a HIP graph."""
    require_gpu(logits, tokens, temperature)
    dev = logits.device
    if elsewhere(dev):
        with torch.cuda.device(dev):
            return token_logprobs(logits, tokens, temperature, top)
    if logits.dim() != 3 or logits.shape[2] < 1:
        raise ValueError("logits must be [B, J, V]")
    if logits.requires_grad and torch.is_grad_enabled():
        raise ValueError("token_logprobs has no gradient: pass logits.detach()")
    if (temperature is not None and temperature.requires_grad
            and torch.is_grad_enabled()):
        raise ValueError("token_logprobs has no gradient: pass "
                         "temperature.detach()")
    b, j, v = logits.shape
    code = _lib.DTYPE_CODES.get(logits.dtype)
    if code is None:
        raise ValueError("logits must be bfloat16, float16 or float32")
    sb, sj, sv = logits.stride()
    if sv != 1 and v > 1:
        raise ValueError("logits must be contiguous along the vocabulary")
    if (tokens.dtype is not torch.int32 or tokens.device != dev
            or tokens.shape != (b, j) or not tokens.is_contiguous()):
        raise ValueError(f"tokens must be a contiguous int32 [{b}, {j}] tensor "
                         f"on {dev}")
    if temperature is not None and (
            temperature.dtype is not torch.float32 or temperature.device != dev
            or temperature.shape != (b,) or not temperature.is_contiguous()):
        raise ValueError(f"temperature must be a contiguous float32 [{b}] "
                         f"tensor on {dev}")
    if not 0 <= top <= _lib.LOGPROBS_TOP:
        raise ValueError(f"top must be in 0..{_lib.LOGPROBS_TOP}")
    logprob, entropy = torch.empty(2, b, j, dtype=torch.float32,
                                   device=dev).unbind(0)
    ids = torch.empty(b, j, top, dtype=torch.int32, device=dev)
    alt = torch.empty(b, j, top, dtype=torch.float32, device=dev)
    out = TokenLogprobs(logprob, entropy, ids, alt)
    if b == 0 or j == 0:
        return out
    L = lib()
    nbytes = _sizes.get((b, j, v, top))
    if nbytes is None:
        nbytes = _sizes[b, j, v, top] = L.sfx_logprobs_workspace_size(b, j, v,
                                                                     top)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    args = _lib.SfxLogprobs(logits.data_ptr(), code, b, j, v, sb, sj,
                            tokens.data_ptr(),
                            None if temperature is None
                            else temperature.data_ptr(),
                            top, logprob.data_ptr(), entropy.data_ptr(),
                            ids.data_ptr() or None, alt.data_ptr() or None)
    check(L.sfx_token_logprobs(args, ws.data_ptr(), nbytes, stream_of(dev)),
          "token_logprobs")
    return out
