"""Speculative decoding with everything on the device: the drafter, a target
model's attention over a cache held in 4 bits, and the verification of the
drafts.

    python examples/speculative_decode.py [--batch 8] [--new 128] [--sample]
                                          [--blocks 0]

The target model is a stand-in of random weights (one attention layer between an
embedding and its transpose); what matters is the loop around it, which is an
engine's:

    propose_with_update   the last step's tokens enter the rows, a draft comes out
    PagePool.resize       pages for the tokens that come, and those back that
                          rejected drafts and finished rows held
    KV4Cache.append       keys and values of the newest token and the draft
    KV4Cache.attend       their queries over the whole cache; with --blocks N
                          .select_blocks and .attend_blocks: over N blocks of 32
                          tokens each
    verify_draft          which drafts stay, and the token after them
    token_logprobs        what is reported of the tokens

No step reads device memory on the host.  A rejected draft's keys and values stay
in the cache until the next append overwrites them.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from suffixgpu_amd import (KV4Cache, PagePool, SuffixGPUDrafter,  # noqa: E402
                           token_logprobs, verify_draft)


class TinyTarget:
    """Embedding -> one attention layer over the 4-bit cache -> logits."""

    def __init__(self, vocab=128, heads=8, kv_heads=2, head_dim=64, seed=0,
                 device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)
        width = heads * head_dim

        def weight(*shape):
            return torch.randn(*shape, generator=g, device=device).mul_(
                shape[0] ** -0.5).to(torch.bfloat16)

        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.embed = weight(width, vocab).t().contiguous()
        self.qkv = weight(width, width + 2 * kv_heads * head_dim)
        self.out = weight(width, width)
        self.lm = weight(width, vocab)
        half = torch.arange(width // 2, device=device)
        self.freq = 0.5 ** (half * (10.0 / half.numel()))

    def forward(self, tokens, start, count, cache, table, blocks=0):
        """Logits [B, T, V] (float32) of tokens [B, T] at positions start + i,
        i < count, which enter the cache; attention over the whole of it, or over
        `blocks` selected blocks."""
        b, t = tokens.shape
        x = self.embed[tokens.clamp(min=0).long()]
        pos = (start[:, None] + torch.arange(t, device=start.device))
        angle = pos[..., None] * self.freq
        x = x + 0.02 * torch.cat([angle.sin(), angle.cos()], -1).to(x.dtype)
        y = (x @ self.qkv).view(b, t, -1, self.head_dim)
        q = y[:, :, :self.heads]
        k = y[:, :, self.heads:self.heads + self.kv_heads]
        v = y[:, :, self.heads + self.kv_heads:]
        cache.append(k, v, table, start, count)
        end = start + count
        if blocks:
            chosen = cache.select_blocks(q, table, end, count, blocks)
            o = cache.attend_blocks(q, chosen, table, end, count)
        else:
            o = cache.attend(q, table, end, count)
        x = x + 0.25 * (o.reshape(b, t, -1) @ self.out)
        return (x @ self.lm).float()


def decode(batch=8, prompt=48, new=128, k=8, vocab=128, temperature=0.0,
           seed=0, device="cuda", draft=True, blocks=0, report=False):
    """Decodes `batch` random prompts until every row has `new` more tokens.
    Returns (rows [batch, prompt + new] of tokens, steps), with `report` also the
    new tokens' log probabilities [batch, new] under the target's logits."""
    dev = torch.device(device, torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    longest = prompt + new + k + 1
    model = TinyTarget(vocab=vocab, seed=seed, device=dev)
    page = 64
    width = -(-longest // page)
    cache = KV4Cache(batch * width, model.kv_heads, model.head_dim,
                     page_size=page, device=dev, bounds=blocks > 0)
    pool = PagePool(batch * width, batch, width, page_size=page, device=dev)
    drafter = SuffixGPUDrafter(k=k, device=dev, max_pattern_len=16,
                               num_backoff=4)
    rows = torch.zeros(batch, longest, dtype=torch.int32, device=dev)
    rows[:, :prompt] = torch.randint(0, vocab, (batch, prompt), generator=g,
                                     device=dev, dtype=torch.int32)
    # the prompts' keys and values, and the first token of every row
    zero = torch.zeros(batch, dtype=torch.int32, device=dev)
    counts = torch.full((batch,), prompt, dtype=torch.int32, device=dev)
    pool.resize(counts)
    logits = model.forward(rows[:, :prompt], zero, counts, cache, pool.table,
                           blocks)
    # (a column behind the rows for what is no token)
    logprobs = torch.zeros(batch, longest + 1, device=dev)

    def note(logits, sampled, start):
        if report:
            at = start[:, None] + torch.arange(sampled.shape[1], device=dev)
            at = torch.where((sampled >= 0) & (at < longest), at, longest)
            logprobs.scatter_(1, at.long(),
                              token_logprobs(logits, sampled).logprob)

    temp = torch.full((batch,), float(temperature), device=dev)

    def verify(logits, drafts, valid):
        kk = drafts.shape[1]
        if temperature == 0:
            return verify_draft(logits, drafts, valid, greedy=True)
        return verify_draft(
            logits, drafts, valid,
            torch.rand(batch, kk, generator=g, device=dev),
            torch.empty(batch, vocab, device=dev).exponential_(generator=g),
            temp)

    none = torch.empty(batch, 0, dtype=torch.int32, device=dev)
    sampled, _ = verify(logits[:, -1:], none, zero)
    note(logits[:, -1:], sampled, counts)
    steps = 0
    # (the host looks at the counts now and then only to know when to stop)
    while True:
        drafts, valid, counts = drafter.propose_with_update(
            counts, rows, sampled, max_model_len=prompt + new)
        if not draft:
            valid = torch.zeros_like(valid)
        if steps % 8 == 0 and int(counts.min()) >= prompt + new:
            done = (rows[:, :prompt + new], steps)
            return (*done, logprobs[:, prompt:prompt + new]) if report else done
        # rows that are done stay where they are
        done = counts >= prompt + new
        valid = torch.where(done, 0, valid)
        counts = counts.clamp(max=prompt + new)
        last = rows.gather(1, (counts - 1).long()[:, None])
        # a row that is done gives its pages back; its token is written nowhere
        pool.resize(torch.where(done, 0, counts + valid))
        logits = model.forward(torch.cat([last, drafts], 1), counts - 1,
                               valid + 1, cache, pool.table, blocks)
        sampled, _ = verify(logits, drafts, valid)
        sampled = torch.where(done[:, None], -1, sampled)
        note(logits, sampled, counts)
        steps += 1


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--new", type=int, default=128)
    ap.add_argument("--sample", action="store_true",
                    help="temperature 0.2 instead of the likeliest token")
    ap.add_argument("--blocks", type=int, default=0,
                    help="attend to so many blocks of 32 tokens (all: 0)")
    a = ap.parse_args()
    t = 0.2 if a.sample else 0.0
    rows, steps, lp = decode(batch=a.batch, new=a.new, temperature=t,
                             blocks=a.blocks, report=True)
    plain, plain_steps = decode(batch=a.batch, new=a.new, temperature=t,
                                draft=False, blocks=a.blocks)
    print(f"{a.new} tokens for {a.batch} requests: {steps} steps with drafts, "
          f"{plain_steps} without; {-lp.mean().item():.2f} nats a token")
    if t == 0:
        same = (rows == plain).float().mean().item()
        print(f"{100 * same:.1f}% of the tokens are the same either way")


if __name__ == "__main__":
    main()
