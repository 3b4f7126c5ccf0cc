"""More operators of the target model's step, as measurable cases.

Families (a case's "do"):

* ``logprobs`` -- token_logprobs: log probabilities of the tokens that
                  verify_draft gave, the entropy they were drawn with, and the
                  likeliest alternatives.
* ``pages``    -- PagePool.resize and PagePool.slots: page tables and slot maps
                  from the requests' lengths, grown for a step's tokens and cut
                  back to what it kept.
* ``sparse``   -- KV4Cache.update_bounds of the newest tokens' blocks, then
                  KV4Cache.select_blocks and KV4Cache.attend_blocks: attention
                  over the blocks of 32 tokens with the largest possible scores.

The cache is the paged one of 4 bits.  A block (32 tokens of a KV head of width D)
holds
  32 x D/2 bytes   keys, token by token, channel 2i in the low half of byte i
  32 x D/32 bytes  their scales 2^(byte - 127), one for 32 channels
  D/64 x 64 x 16   values: 32-bit words of 8 tokens of one channel, word
                   [c // 64][2s + h][c % 16][c // 16 % 4] holding in its j-th
                   four bits token 16 s + 8 (j // 4) + 4 h + j % 4
  32 x 4 bytes     their float32 scales, one a token
The four bits are a sign and one of 0, .5, 1, 1.5, 2, 3, 4, 6.

Of a block's keys the bounds are, per channel, the least and the largest in whole
units of 2^u, rounded outwards, with 2^(u + 6) the power of two at or below the
largest magnitude of all.  A query token scores a block, per KV head, by
  2^u sum_c (P_c hi_c - N_c lo_c)
with P and N the sums over the head's query heads of the positive and of the
negated negative channels, rounded to 7 bits: the largest that the sum of their
products with one of the block's keys can be.  It takes the first blocks and the
most recent ones, then those with the largest scores, the lowest on ties.
"""

import math
import random

import torch

own = False

DEV = "cuda"
VOCAB = 128256
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
INF = math.inf
FIRST, RECENT = 1, 2      # blocks that a query always takes


# ------------------------------------------------------------------ cases
def _logprobs(name, b, j, v, dtype, top, temp="one", pad=0, ragged=True):
    return {"name": name, "do": "logprobs", "b": b, "j": j, "v": v,
            "dtype": dtype, "top": top, "temp": temp, "pad": pad,
            "ragged": ragged}


def _pages(name, rows, page, ctx, new, turn=0.0, supply=1.2):
    return {"name": name, "do": "pages", "rows": rows, "page": page,
            "ctx": ctx, "new": new, "turn": turn, "supply": supply}


def _sparse(name, b, t, hq, hkv, d, dtype, ctx, blocks, page=64, fill=0.5,
            ragged=True):
    return {"name": name, "do": "sparse", "b": b, "t": t, "hq": hq,
            "hkv": hkv, "d": d, "dtype": dtype, "ctx": ctx, "blocks": blocks,
            "page": page, "fill": fill, "ragged": ragged}


def listed():
    return [
        # One chat request's newest token, with five alternatives.
        _logprobs("logprobs_b1_j1_v32000_f32", 1, 1, 32000, "f32", 5),
        # The headline decode step: what 64 verified drafts of 16 kept, as many
        # as each has.
        _logprobs("logprobs_b64_j17_v128256", 64, 17, VOCAB, "bf16", 5),
        # A large server without drafts, temperatures of its requests' own, as
        # many alternatives as interfaces offer.
        _logprobs("logprobs_b256_j1_top20", 256, 1, VOCAB, "bf16", 20,
                  temp="mixed"),
        # An odd vocabulary whose rows start at any alignment, no alternatives.
        _logprobs("logprobs_b16_j8_v65003_f16", 16, 8, 65003, "f16", 0,
                  temp="mixed"),
        # The tokens of a prompt's chunk under the model that read it.
        _logprobs("logprobs_prompt_j2048", 1, 2048, VOCAB, "bf16", 1,
                  ragged=False),
        # The headline step: room for a token and 16 drafts, cut back again.
        _pages("pages_r64_new17", 64, 64, 8192, 17),
        # Requests come and go, prompts' chunks enter, and pages run short.
        _pages("pages_r256_new4096_turn", 256, 32, 65536, 4096, turn=0.25,
               supply=0.7),
        # One chat request's single token over a long history.
        _sparse("sparse_b1_t1_s131072", 1, 1, 32, 8, 128, "bf16", 131072, 128,
                fill=1.0),
        # A decode step without drafts: 64 requests of up to 32768 tokens.
        _sparse("sparse_b64_t1_s32768", 64, 1, 32, 8, 128, "bf16", 32768, 64),
        # The headline step's verification: up to 16 drafts a request.
        _sparse("sparse_b64_t17_s8192", 64, 17, 32, 8, 128, "bf16", 8192, 32),
        # A few long documents, wide heads, small groups.
        _sparse("sparse_b4_t9_s131072_d256_f16", 4, 9, 16, 8, 256, "f16",
                131072, 96, page=256, fill=0.9),
        # A chunk of a long prompt.
        _sparse("sparse_prompt_t2048_s16384", 1, 2048, 32, 8, 128, "bf16",
                16384, 64, fill=1.0, ragged=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case; its cost is bounded by the largest listed one's."""
    do = rng.choice(("logprobs", "logprobs", "pages", "sparse", "sparse",
                     "sparse"))
    while True:
        if do == "logprobs":
            c = _logprobs("", _log_int(rng, 1, 256), _log_int(rng, 1, 64),
                          _log_int(rng, 30000, 132000),
                          rng.choice(("bf16", "bf16", "f16", "f32")),
                          rng.choice((0, 1, 5, 8, 20, 31)),
                          temp=rng.choice(("one", "mixed")),
                          pad=rng.choice((0, 0, 1, 56)),
                          ragged=rng.random() < 0.6)
            ok = c["b"] * c["j"] * c["v"] <= 2048 * VOCAB // (
                2 if c["dtype"] == "f32" else 1)
        elif do == "pages":
            new = _log_int(rng, 1, 4200)
            c = _pages("", _log_int(rng, 1, 256), rng.choice((32, 64, 128, 256)),
                       new + _log_int(rng, 64, 60000), new,
                       turn=rng.choice((0.0, 0.1, 0.5)),
                       supply=rng.choice((0.4, 1.0, 1.5)))
            ok = c["rows"] * c["ctx"] // c["page"] <= 256 * 2048
        else:
            hkv = rng.choice((1, 2, 4, 8))
            t = _log_int(rng, 1, 600)
            c = _sparse("", _log_int(rng, 1, 128), t,
                        hkv * rng.choice((1, 2, 3, 4, 5, 8)), hkv,
                        rng.choice((64, 128, 256)),
                        rng.choice(("bf16", "f16")),
                        t + _log_int(rng, 32, 131072),
                        _log_int(rng, 4, 200),
                        page=rng.choice((32, 64, 128, 256)),
                        fill=rng.choice((0.1, 0.5, 0.95)),
                        ragged=rng.random() < 0.6)
            lists = c["b"] * t * hkv
            ok = (c["b"] * c["ctx"] * hkv * c["d"] <= 64 * 32768 * 8 * 128
                  and lists * c["blocks"] * c["d"] <= 2048 * 8 * 64 * 128
                  and lists * c["ctx"] <= 2048 * 8 * 16384)
        if ok:
            del c["name"]
            return c


# A case's lengths belong to the case: every seed has the same.
def _rng_of(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items()
                                     if k != "name")))


def _kept(case):
    """Tokens per request that have a log probability."""
    r = _rng_of(case)
    return [r.randint(1, case["j"]) if case["ragged"] else case["j"]
            for _ in range(case["b"])]


def _page_lens(case):
    """Lengths before a step, with a step's tokens, and those tokens' number."""
    r = _rng_of(case)
    before, after, new = [], [], []
    for _ in range(case["rows"]):
        n = r.randint(1, case["new"])
        a = r.randint(0, case["ctx"] - n)
        b = a + n
        if r.random() < case["turn"]:
            # a request ends here, or another one takes its row
            b = r.choice((0, r.randint(n, case["ctx"])))
            n = min(n, b)
        before.append(a)
        after.append(b)
        new.append(n)
    return before, after, new


def _page_count(case):
    """Pages of the pool: some more, or less, than the step needs."""
    before, after, _ = _page_lens(case)
    p = case["page"]
    held = [-(-a // p) for a in before]
    grow = sum(max(0, -(-b // p) - h) for b, h in zip(after, held))
    return sum(held) + int(case["supply"] * grow)


def _new_tokens(case):
    r = _rng_of(case)
    return [r.randint(1, case["t"]) if case["ragged"] else case["t"]
            for _ in range(case["b"])]


def _kv_lens(case):
    r = _rng_of(case)
    n = _new_tokens(case)
    lo = int(case["fill"] * case["ctx"])
    return [max(m, r.randint(lo, case["ctx"])) for m in n]


def work(case):
    if case["do"] == "logprobs":
        w = 4 if case["dtype"] == "f32" else 2
        rows = sum(_kept(case))
        out = case["b"] * case["j"] * (12 + 8 * case["top"])
        return {"bytes": float(rows * case["v"] * w + out),
                "flops": float(rows * case["v"] * 6)}
    if case["do"] == "pages":
        before, after, new = _page_lens(case)
        p = case["page"]
        moved = sum(abs(-(-b // p) + a // -p) for a, b in zip(before, after))
        # the step's tokens' slots and pages, and each page that comes or goes
        # from one list to the other, there and back
        return {"bytes": float(case["rows"] * (28 + 8 * case["new"])
                               + sum(4 * -(-n // p) for n in new)
                               + 16 * moved),
                "flops": 0.0}
    d, hkv, g = case["d"], case["hkv"], case["hq"] // case["hkv"]
    tok = 2 * (d // 2) + d // 32 + 4          # a token of a KV head
    bytes_ = flops = 0
    for n, ln in zip(_new_tokens(case), _kv_lens(case)):
        seen = -(-ln // 32)
        took = taken = 0
        for i in range(n):
            own_blocks = -(-(ln - n + i + 1) // 32)
            took = min(case["blocks"], own_blocks)
            taken += took
            flops += hkv * (4 * d * own_blocks + took * 32 * 4 * d * g)
        # blocks that some query takes: at least the last one's
        bytes_ += hkv * (seen * (2 * d + 1) + took * 32 * tok + 4 * taken)
        # the new tokens' blocks, whose bounds follow them
        touched = (ln - 1) // 32 - (ln - n) // 32 + 1
        bytes_ += hkv * touched * 32 * (d // 2 + d // 32)
        bytes_ += 4 * case["hq"] * d * n
    return {"bytes": float(bytes_), "flops": float(flops)}


# ----------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _ints(xs):
    return torch.tensor(xs, dtype=torch.int32, device=DEV)


def _prepare_logprobs(case, seed):
    g = _gen(seed)
    b, j, v = case["b"], case["j"], case["v"]
    buf = torch.empty(b, j, v + case["pad"], dtype=DTYPES[case["dtype"]],
                      device=DEV)
    for i in range(b):
        buf[i] = torch.randn(j, v + case["pad"], generator=g, device=DEV) * 2.5
    logits = buf[..., :v]
    # mostly a likely token, sometimes any, as sampling gives
    tokens = torch.randint(0, v, (b, j), generator=g, device=DEV)
    likely = torch.rand(b, j, generator=g, device=DEV) < 0.8
    boost = torch.rand(b, j, generator=g, device=DEV) * 6 + 10
    at = tokens[..., None]
    old = logits.gather(2, at)
    logits.scatter_(2, at, torch.where(likely[..., None],
                                       boost[..., None].to(buf.dtype), old))
    tokens[torch.arange(j, device=DEV) >= _ints(_kept(case))[:, None]] = -1
    temp = None
    if case["temp"] == "mixed":
        temp = torch.rand(b, generator=g, device=DEV) * 0.6 + 0.6
        temp[3::4] = 0.0
    return {"case": case, "logits": logits, "tokens": tokens.int(),
            "temperature": temp, "top": case["top"]}


def _prepare_pages(case, seed):
    before, after, new = _page_lens(case)
    width = -(-case["ctx"] // case["page"])
    n, rows = _page_count(case), case["rows"]
    g = _gen(seed)
    # the rows' pages come from requests that were here before
    past = torch.randint(0, case["ctx"] + 1, (rows,), generator=g, device=DEV,
                         dtype=torch.int32)
    st = {"case": case, "before": _ints(before), "after": _ints(after),
          "new": _ints(new),
          "start": _ints([b - m for b, m in zip(after, new)])}
    if own:
        from suffixgpu_amd import PagePool
        st["pool"] = PagePool(n, rows, width, page_size=case["page"],
                              device=DEV)
        st["pool"].resize(past)
        st["pool"].resize(st["before"])
        st["pool"].resize(st["before"])
        return st
    # (the last entry of the stack is no page's: what moves nowhere goes there)
    stack = torch.arange(n, -1, -1, dtype=torch.int32, device=DEV)
    stack = torch.cat([stack[1:], stack[:1]])
    st["pool"] = {"page": case["page"], "stack": stack,
                  "free": torch.full((), n, dtype=torch.int64, device=DEV),
                  "held": torch.zeros(rows, dtype=torch.int64, device=DEV),
                  "table": torch.full((rows, width), -1, dtype=torch.int32,
                                      device=DEV)}
    _resize_plain(st["pool"], past)
    _resize_plain(st["pool"], st["before"])
    _resize_plain(st["pool"], st["before"])
    return st


def _block_bytes(d):
    return 32 * (d // 2) + 32 * (d // 32) + 32 * (d // 2) + 128


def _random_pages(case, n, g):
    """A pool whose four-bit values are rounded normal numbers, scales of the
    size that such keys and values have; some blocks hold larger keys."""
    d, blocks = case["d"], n * case["hkv"] * (case["page"] // 32)
    q = torch.erfinv(torch.linspace(-1, 1, 258, dtype=torch.float64)[1:-1]
                     ) * math.sqrt(2.0) * 2.0
    mid = torch.tensor([.25, .75, 1.25, 1.75, 2.5, 3.5, 5.],
                       dtype=torch.float64)
    code = torch.bucketize(q.abs(), mid) + 8 * (q < 0)
    both = (code[:, None] | (code[None, :] << 4)).to(torch.uint8).reshape(-1)
    both = both.to(DEV)
    pages = torch.empty(blocks, _block_bytes(d), dtype=torch.uint8,
                        device=DEV)
    ks, vw = 16 * d, 17 * d
    step = max(1, (1 << 25) // d)
    for i in range(0, blocks, step):
        m = min(step, blocks - i)
        r = torch.randint(0, 1 << 16, (m, 32 * d), generator=g, device=DEV,
                          dtype=torch.int32)
        r = both[r]
        p = pages[i:i + m]
        p[:, :ks] = r[:, :ks]
        p[:, vw:vw + 16 * d] = r[:, ks:]
        e = torch.randint(125, 127, (m, d), generator=g, device=DEV,
                          dtype=torch.int32)
        e += torch.rand(m, 1, generator=g, device=DEV) < 0.1
        p[:, ks:vw] = e.to(torch.uint8)
        s = torch.rand(m, 32, generator=g, device=DEV) * 0.4 + 0.2
        p[:, vw + 16 * d:] = s.view(torch.uint8)
    return pages.view(n, case["hkv"], case["page"] // 32, -1)


def _prepare_sparse(case, seed):
    g = _gen(seed)
    width = -(-case["ctx"] // case["page"])
    n = case["b"] * width
    table = torch.randperm(n, generator=g, device=DEV).to(torch.int32)
    table = table.view(case["b"], width)
    pages = _random_pages(case, n, g)
    hkv = case["hkv"]
    # query, key and value heads as a model's one projection gives them
    x = torch.randn(case["b"], case["t"], case["hq"] + 2 * hkv, case["d"],
                    generator=g, device=DEV)
    x = x.mul_(1.5).to(DTYPES[case["dtype"]])
    new, lens = _new_tokens(case), _kv_lens(case)
    st = {"case": case, "table": table, "pages": pages, "new": _ints(new),
          "kv_len": _ints(lens), "q": x[:, :, :case["hq"]],
          "start": _ints([a - m for a, m in zip(lens, new)])}
    if own:
        # the tokens before the newest have their bounds from earlier calls
        from suffixgpu_amd import KV4Cache
        st["cache"] = KV4Cache(n, hkv, case["d"], page_size=case["page"],
                               dtype=DTYPES[case["dtype"]], device=DEV,
                               pages=pages, bounds=True)
        st["cache"].update_bounds(table, _ints([0] * case["b"]), max(lens),
                                  _ints(lens))
        return st
    # lo, hi [pages, heads, blocks, D] and the units
    flat = pages.view(-1, pages.shape[-1])
    step = max(1, (1 << 22) // case["d"])
    got = [_bounds_plain(flat[i:i + step], case["d"], None)
           for i in range(0, flat.shape[0], step)]
    st["bounds"] = [torch.cat(y).view(*pages.shape[:3], -1)
                    for y in zip(*got)]
    return st


def prepare(case, seed):
    if case["do"] == "logprobs":
        return _prepare_logprobs(case, seed)
    if case["do"] == "pages":
        return _prepare_pages(case, seed)
    return _prepare_sparse(case, seed)


# ------------------------------------------------------------ plain forms
def _logprobs_plain(s):
    x, tok, n = s["logits"].float(), s["tokens"].long(), s["top"]
    b, j, v = x.shape
    x = torch.where(torch.isnan(x), -INF, x) + 0.0
    t = s["temperature"]
    t = torch.ones(b, device=x.device) if t is None else t
    t = t[:, None, None]
    greedy = ~(t > 0)
    col = torch.arange(v, device=x.device)
    given = (tok >= 0) & (tok < v)
    top = x.amax(dim=2, keepdim=True)
    some = given[..., None] & (top > -INF)
    arg = torch.where(x == top, col, v).amin(dim=2, keepdim=True)
    z = torch.where(x == top, 0.0, x - top) / torch.where(greedy, 1.0, t)
    z = torch.where(greedy, torch.where(col == arg, 0.0, -INF), z)
    e = torch.exp(z)
    # in 64 bits: a likely token's log probability is what the others add to one
    total = e.sum(dim=2, dtype=torch.float64)
    log = torch.log(total)
    entropy = torch.where(z > -INF, z * e, 0.0).sum(dim=2, dtype=torch.float64)
    entropy = torch.where(some[..., 0], log - entropy / total, 0.0).float()

    def of(at):
        lp = z.gather(2, at).double() - log[..., None]
        return torch.where(some, lp, -INF).float()

    logprob = of(tok.clamp(0, v - 1)[..., None])[..., 0]
    logprob = torch.where(given, logprob, 0.0)
    # whole numbers that rank as the logits do, the lowest index first
    bits = x.view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long()
    best = torch.topk((bits << 32) + (0x7fffffff - col), n, dim=2).indices
    there = some & (x.gather(2, best) > -INF)
    return (logprob, entropy, torch.where(there, best, -1).int(),
            torch.where(there, of(best), -INF))


def _resize_plain(p, lengths):
    page, stack, held, table = p["page"], p["stack"], p["held"], p["table"]
    rows, width = table.shape
    want = torch.clamp((lengths.long() + page - 1) // page, max=width)
    want = torch.where(lengths < 0, held, want)
    need = (want - held).clamp(min=0)
    back = (held - want).clamp(min=0)
    got = (p["free"] - (need.cumsum(0) - need)).clamp(min=0)
    got = torch.minimum(got, need)
    left = p["free"] - got.sum()
    at = torch.arange(width, device=table.device)
    dummy = stack.shape[0] - 1
    # the i-th page taken is the i-th from the top
    i = (got.cumsum(0) - got)[:, None] + at - held[:, None]
    take = (at >= held[:, None]) & (at < (held + got)[:, None])
    taken = stack[torch.where(take, p["free"] - 1 - i, dummy)]
    # of the pages that come back the first row's first ends on top
    i = (back.sum() - back.cumsum(0))[:, None] + held[:, None] - 1 - at
    gone = (at >= want[:, None]) & (at < held[:, None])
    stack[torch.where(gone, left + i, dummy)] = table
    table.copy_(torch.where(take, taken, torch.where(gone, -1, table)))
    held.copy_(torch.where(back > 0, want, held + got))
    p["free"] = left + back.sum()
    return (held * page).int()


def _pages_plain(s):
    p = s["pool"]
    page, width = p["page"], p["table"].shape[1]
    room = _resize_plain(p, s["after"])
    i = torch.arange(s["case"]["new"], device=DEV)
    pos = s["start"][:, None].long() + i
    ok = (i < s["new"][:, None]) & (pos < width * page)
    at = torch.where(ok, pos // page, 0)
    ids = p["table"].gather(1, at).long()
    slots = torch.where(ok & (ids >= 0), ids * page + pos % page, -1)
    table = p["table"].clone()
    _resize_plain(p, s["before"])
    return room, slots, table, p["held"].int()


def _unpack_k(blk, d):
    """[n, block bytes] -> keys [n, 32, d] float32."""
    n = blk.shape[0]
    lut = torch.tensor(E2M1 + tuple(-x for x in E2M1), device=blk.device)
    c = blk[:, :16 * d].reshape(n, 32, d // 2)
    k = lut[torch.stack((c & 15, c >> 4), dim=-1).int()]
    sc = torch.exp2(blk[:, 16 * d:17 * d].float() - 127)
    return (k.view(n, 32, d // 32, 32)
            * sc.view(n, 32, d // 32, 1)).view(n, 32, d)


def _unpack_v(blk, d):
    n, vw = blk.shape[0], 17 * d
    lut = torch.tensor(E2M1 + tuple(-x for x in E2M1), device=blk.device)
    c = blk[:, vw:vw + 16 * d].reshape(n, d // 64, 2, 2, 16, 4, 4)
    c = torch.stack((c & 15, c >> 4), dim=-1).int()
    # [n, group, s, h, channel, tile, (a, r)] -> tokens (s, a, h, r)
    c = c.view(n, d // 64, 2, 2, 16, 4, 2, 4).permute(0, 2, 6, 3, 7, 1, 5, 4)
    sv = blk[:, vw + 16 * d:].contiguous().view(torch.float32).view(n, 32, 1)
    return lut[c.reshape(n, 32, d)] * sv


def _bounds_plain(blk, d, count):
    """Least and largest key per channel of [n, block bytes], in units of 2^u,
    and u; count: tokens of each block, all without it."""
    k = _unpack_k(blk, d)
    hi, lo = k, k
    if count is not None:
        there = torch.arange(32, device=blk.device) < count[:, None]
        hi = torch.where(there[..., None], k, -INF)
        lo = torch.where(there[..., None], k, INF)
    hi, lo = hi.amax(dim=1), lo.amin(dim=1)
    top = torch.maximum(hi.abs(), lo.abs()).amax(dim=1, keepdim=True)
    _, e = torch.frexp(top)                   # top = f 2^e, .5 <= f < 1
    u = torch.where(top > 0, (e - 7).clamp(-100, 100), -100)
    hi = torch.ceil(torch.ldexp(hi, -u)).clamp(-127, 127)
    lo = torch.floor(torch.ldexp(lo, -u)).clamp(-127, 127)
    return lo.to(torch.int8), hi.to(torch.int8), u.to(torch.int8)


def _update_plain(s):
    """The bounds of the blocks that hold the newest tokens."""
    case = s["case"]
    d, page = case["d"], case["page"]
    per = page // 32
    most = (case["t"] + 30) // 32 + 1
    end = s["start"].long() + s["new"]
    blk = (s["start"].long() // 32)[:, None] + torch.arange(most, device=DEV)
    # where a row touches fewer blocks: the last of them again
    blk = torch.minimum(blk, ((end - 1) // 32)[:, None])
    ids = s["table"].long().gather(1, blk // per)
    at = (ids[..., None] * case["hkv"]
          + torch.arange(case["hkv"], device=DEV)) * per
    at = (at + (blk % per)[..., None]).reshape(-1)
    count = (end[:, None] - blk * 32).clamp(max=32)
    count = count[..., None].expand(-1, -1, case["hkv"]).reshape(-1)
    got = _bounds_plain(s["pages"].view(-1, s["pages"].shape[-1])[at], d,
                        count)
    for x, y in zip(s["bounds"], got):
        x.view(-1, x.shape[-1])[at] = y


def _select_plain(s):
    """Block ids [b, t, hkv, blocks] in order, -1 behind them."""
    case = s["case"]
    b, t, hq, d = s["q"].shape
    hkv, n = case["hkv"], case["blocks"]
    q = s["q"].float().view(b, t, hkv, hq // hkv, d)
    _, e = torch.frexp(q.abs().amax(dim=(3, 4), keepdim=True))
    q = torch.round(torch.ldexp(q, 15 - e)).long()
    p = torch.cat([(-q).clamp(min=0).sum(dim=3), q.clamp(min=0).sum(dim=3)],
                  dim=-1)                            # against lo, against hi
    top = p.amax(dim=-1, keepdim=True)
    _, bits = torch.frexp(top.double())              # top < 2^bits
    shift = (bits.long() - 7).clamp(min=0)
    p = ((p + ((1 << shift) >> 1)) >> shift).clamp(max=127)
    p[..., :d] *= -1
    out = []
    for i in range(b):
        lo, hi, u = (x[s["table"][i].long()].transpose(0, 1)
                     .reshape(hkv, -1, x.shape[-1]) for x in s["bounds"])
        m = lo.shape[1]
        lh = torch.cat([lo, hi], dim=-1).float()
        # whole numbers below 2^24: exact in 32 bits
        w = torch.matmul(p[i].transpose(0, 1).float(), lh.transpose(1, 2))
        w = torch.ldexp(w.double(), u.view(hkv, 1, m).int()).transpose(0, 1)
        pos = s["start"][i] + torch.arange(t, device=DEV)
        last = torch.where(torch.arange(t, device=DEV) < s["new"][i],
                           pos // 32, -1)[:, None, None]
        j = torch.arange(m, device=DEV)
        w = torch.where((j < FIRST) | (j > last - RECENT), INF, w)
        w = torch.where(j <= last, w, -INF)
        order = torch.argsort(w, dim=-1, descending=True, stable=True)
        order = order[..., :n]
        order = torch.where(order <= last, order, m)
        order = order.sort(dim=-1).values
        order = torch.where(order < m, order, -1)
        out.append(torch.nn.functional.pad(order, (0, n - order.shape[-1]),
                                           value=-1))
    return torch.stack(out).int()


def _attend_plain(s, sel):
    case = s["case"]
    b, t, hq, d = s["q"].shape
    hkv, n, page = case["hkv"], case["blocks"], case["page"]
    g, per = hq // hkv, page // 32
    sel = sel.long().view(-1, n)                         # a list a row
    of = torch.arange(b * t * hkv, device=DEV)
    row, tok, head = of // (t * hkv), of // hkv % t, of % hkv
    q = s["q"].reshape(b * t * hkv, g, d)
    flat = s["pages"].view(-1, s["pages"].shape[-1])
    pos = s["start"].long()[row] + tok
    out = torch.zeros(b * t * hkv, g, d, dtype=s["q"].dtype, device=DEV)
    step = max(1, (1 << 22) // (n * d))
    for i in range(0, b * t * hkv, step):
        x, r = sel[i:i + step], row[i:i + step]
        ids = s["table"][r[:, None], x.clamp(min=0) // per].long()
        at = (ids * hkv + head[i:i + step, None]) * per + x.clamp(min=0) % per
        blk = flat[at.view(-1)]
        k = _unpack_k(blk, d).view(-1, n * 32, d)
        w = torch.matmul(q[i:i + step].float(), k.transpose(1, 2))
        w = w * (1.0 / math.sqrt(d))
        p = x[..., None] * 32 + torch.arange(32, device=DEV)
        see = (x[..., None] >= 0) & (p <= pos[i:i + step, None, None])
        see &= (tok[i:i + step] < s["new"][r])[:, None, None]
        w = torch.where(see.view(-1, 1, n * 32), w, -INF)
        m = w.amax(dim=-1, keepdim=True)
        w = torch.exp(w - torch.where(m == -INF, 0.0, m))
        z = w.sum(dim=-1, keepdim=True)
        o = torch.matmul(w, _unpack_v(blk, d).view(-1, n * 32, d))
        out[i:i + step] = (o / torch.where(z == 0, 1.0, z)).to(out.dtype)
    return out.view(b, t, hq, d)


def run(s):
    do = s["case"]["do"]
    if do == "logprobs":
        if not own:
            return _logprobs_plain(s)
        from suffixgpu_amd import token_logprobs
        return tuple(token_logprobs(s["logits"], s["tokens"],
                                    temperature=s["temperature"],
                                    top=s["top"]))
    if do == "pages":
        if not own:
            return _pages_plain(s)
        pool = s["pool"]
        room = pool.resize(s["after"])
        slots = pool.slots(s["start"], s["case"]["new"], s["new"])
        table = pool.table.clone()
        pool.resize(s["before"])
        return room, slots, table, pool.held
    if not own:
        _update_plain(s)
        sel = _select_plain(s)
        return sel, _attend_plain(s, sel)
    cache, table = s["cache"], s["table"]
    cache.update_bounds(table, s["start"], s["case"]["t"], s["new"])
    sel = cache.select_blocks(s["q"], table, s["kv_len"], s["new"],
                              blocks=s["case"]["blocks"], first=FIRST,
                              recent=RECENT)
    return sel, cache.attend_blocks(s["q"], sel, table, s["kv_len"], s["new"])


# ------------------------------------------------- definitions in 64 bits
def _exact_logprobs(s):
    """Request by request; positions without a token are left as they are said
    to be."""
    b, j, v = s["logits"].shape
    n = s["top"]
    lp = torch.zeros(b, j, dtype=torch.float64, device=DEV)
    h = torch.zeros_like(lp)
    ids = torch.full((b, j, n), -1, dtype=torch.int32, device=DEV)
    alt = torch.full((b, j, n), -INF, dtype=torch.float64, device=DEV)
    kept = _kept(s["case"])
    for i in range(b):
        for a in range(0, kept[i], 64):
            e = min(a + 64, kept[i])
            x = s["logits"][i, a:e].double()
            order = x.sort(dim=1, descending=True, stable=True).indices
            t = 1.0 if s["temperature"] is None else float(s["temperature"][i])
            if t > 0:
                z = torch.log_softmax(x / t, dim=1)
            else:
                z = torch.full_like(x, -INF).scatter_(1, order[:, :1], 0.0)
            lp[i, a:e] = z.gather(1, s["tokens"][i, a:e].long()[:, None])[:, 0]
            h[i, a:e] = torch.special.entr(torch.exp(z)).sum(dim=1)
            ids[i, a:e] = order[:, :n].int()
            alt[i, a:e] = z.gather(1, order[:, :n])
    return lp, h, ids, alt


def _exact_pages(case, seed):
    """Page by page on the host."""
    before, after, new = _page_lens(case)
    page, rows = case["page"], case["rows"]
    width = -(-case["ctx"] // page)
    past = torch.randint(0, case["ctx"] + 1, (rows,), generator=_gen(seed),
                         device=DEV, dtype=torch.int32).tolist()
    free = list(range(_page_count(case) - 1, -1, -1))
    held = [[] for _ in range(rows)]

    def resize(lens):
        back = []
        for r, n in enumerate(lens):
            want = -(-n // page)
            while len(held[r]) < want and free:
                held[r].append(free.pop())
            back += held[r][want:]
            del held[r][want:]
        free.extend(reversed(back))

    for lens in (past, before, before, after):
        resize(lens)
    table = [h + [-1] * (width - len(h)) for h in held]
    room = [len(h) * page for h in held]
    slots = []
    for r in range(rows):
        at = [-1] * case["new"]
        for i in range(new[r]):
            p = after[r] - new[r] + i
            if p < room[r]:
                at[i] = held[r][p // page] * page + p % page
        slots.append(at)
    resize(before)
    return (_ints(room), torch.tensor(slots, dtype=torch.int64), _ints(table),
            _ints([len(h) for h in held]))


def _exact_sparse(s):
    """Row by row and KV head by KV head."""
    case = s["case"]
    d, hkv, page, n = case["d"], case["hkv"], case["page"], case["blocks"]
    b, t, hq, _ = s["q"].shape
    g = hq // hkv
    tok = torch.arange(32, device=DEV)[:, None]
    ch = torch.arange(d, device=DEV)[None, :]
    kb = tok * (d // 2) + ch // 2
    ksh = (4 * (ch % 2)).expand(32, d)
    sb = 16 * d + tok * (d // 32) + ch // 32
    quad = 2 * (tok // 16) + tok // 4 % 2
    j = 4 * (tok // 8 % 2) + tok % 4
    word = ((ch // 64 * 4 + quad) * 16 + ch % 16) * 4 + ch // 16 % 4
    vb = 17 * d + word * 4 + j // 2
    vsh = (4 * (j % 2)).expand(32, d)
    mag = torch.tensor(E2M1, dtype=torch.float64, device=DEV)

    def val(c):
        return torch.where(c >= 8, -1.0, 1.0) * mag[(c & 7).long()]

    sel = torch.full((b, t, hkv, n), -1, dtype=torch.int32, device=DEV)
    out = torch.zeros(b, t, hq, d, dtype=torch.float64, device=DEV)
    lens, new = s["kv_len"].tolist(), s["new"].tolist()
    for i in range(b):
        ids = s["table"][i, :-(-lens[i] // page)].long()
        for h in range(hkv):
            m = -(-lens[i] // 32)
            blk = s["pages"][ids, h].reshape(-1, _block_bytes(d))[:m]
            k = val((blk[:, kb] >> ksh) & 15)
            k = k * 2.0 ** (blk[:, sb].double() - 127)
            sv = blk[:, -128:].contiguous().view(torch.float32).double()
            v = val((blk[:, vb] >> vsh) & 15) * sv[..., None]
            top = k.abs().amax(dim=(1, 2)).clamp(min=2.0 ** -94)
            unit = torch.exp2(torch.floor(torch.log2(top)) - 6)[:, None]
            hi = torch.ceil(k.amax(dim=1) / unit) * unit
            lo = torch.floor(k.amin(dim=1) / unit) * unit
            for r in range(0, new[i], 64):
                e = min(r + 64, new[i])
                q = s["q"][i, r:e, h * g:(h + 1) * g].double()
                f = 2.0 ** (14 - torch.floor(torch.log2(
                    q.abs().amax(dim=(1, 2), keepdim=True))))
                z = torch.round(q * f)
                p = z.clamp(min=0).sum(dim=1)
                w = (-z).clamp(min=0).sum(dim=1)
                a = torch.maximum(p.amax(dim=1), w.amax(dim=1))[:, None]
                # halves up, to numbers of 7 bits
                f = 2.0 ** (torch.floor(torch.log2(a)) - 6).clamp(min=0)
                p = torch.floor(p / f + 0.5).clamp(max=127)
                w = torch.floor(w / f + 0.5).clamp(max=127)
                score = torch.matmul(p, hi.t()) - torch.matmul(w, lo.t())
                last = (lens[i] - new[i] + r
                        + torch.arange(e - r, device=DEV))[:, None]
                at = torch.arange(m, device=DEV)
                score[:, :FIRST] = INF
                score = score.masked_fill(at > last // 32 - RECENT, INF)
                score = score.masked_fill(at > last // 32, -INF)
                best = score.sort(dim=1, descending=True, stable=True)
                took = torch.zeros(e - r, m, dtype=torch.bool, device=DEV)
                took.scatter_(1, best.indices[:, :n],
                              best.values[:, :n] > -INF)
                rank = took.long().cumsum(dim=1) - 1
                where = took.nonzero()
                sel[i, r + where[:, 0], h, rank[took]] = where[:, 1].int()
                see = took.repeat_interleave(32, dim=1)
                see &= torch.arange(m * 32, device=DEV) <= last
                x = torch.matmul(q.reshape(-1, d), k.view(-1, d).t())
                x = (x / math.sqrt(d)).view(e - r, g, -1)
                x = x.masked_fill(~see[:, None], -INF).view(-1, m * 32)
                x = torch.matmul(torch.softmax(x, dim=1), v.view(-1, d))
                out[i, r:e, h * g:(h + 1) * g] = x.view(e - r, g, d)
    return sel, out


def exact(case, seed):
    if case["do"] == "pages":
        return _exact_pages(case, seed)
    if case["do"] == "logprobs":
        return _exact_logprobs(prepare(case, seed))
    return _exact_sparse(prepare(case, seed))
