"""The operators on the target model's side of a step, by their definitions, in
numpy and 64 bits: verification of drafts, log probabilities, page tables, the
rounding of keys and values to 4 bits, and attention over what they then stand for,
all of it or selected blocks."""

from __future__ import annotations

import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def verify(logits, draft, num_valid, uniform, noise, temperature,
           draft_probs=None, margin=2.0 ** -15):
    """(sampled, count, clear): clear[b] is False where a decision of row b is
    nearer than `margin` (relative), so that arithmetic in 32 bits may take
    either side."""
    b, k1, v = logits.shape
    k = k1 - 1
    sampled = np.full((b, k1), -1, dtype=np.int32)
    count = np.zeros(b, dtype=np.int32)
    clear = np.ones(b, dtype=bool)
    for i in range(b):
        n = 0
        while (n < min(int(num_valid[i]), k) and 0 <= draft[i, n] < v):
            n += 1
        t = float(temperature[i]) if temperature is not None else 1.0
        greedy = not t > 0
        for j in range(n + 1):
            x = logits[i, j].astype(np.float64)
            x = np.where(np.isnan(x), -np.inf, x)
            top = x.max()
            if top == -np.inf:
                break
            if greedy:
                tok = int(np.argmax(x))
                sampled[i, j] = tok
                count[i] = j + 1
                if j < n and draft[i, j] == tok:
                    continue
                break
            with np.errstate(invalid="ignore", over="ignore"):
                z = np.where(x == top, 0.0, (x - top) / t)
            p = np.exp(z)
            p /= p.sum()
            r = p
            if j < n:
                d = int(draft[i, j])
                if draft_probs is None:
                    q = np.zeros(v)
                    q[d] = 1.0
                else:
                    q = draft_probs[i, j].astype(np.float64)
                lhs, rhs = float(uniform[i, j]) * q[d], p[d]
                if abs(lhs - rhs) <= margin * max(lhs, rhs):
                    clear[i] = False
                if lhs < rhs:
                    sampled[i, j] = d
                    count[i] = j + 1
                    continue
                r = np.maximum(p - q, 0.0)
                if not (r > 0).any():
                    r = p
            race = r / noise[i].astype(np.float64)
            tok = int(np.argmax(race))
            # a difference p - q carries the error of p
            slack = margin * (race + p / noise[i])
            rest = np.delete(race + slack, tok)
            if rest.size and (rest >= race[tok] - slack[tok]).any():
                clear[i] = False
            sampled[i, j] = tok
            count[i] = j + 1
            break
    return sampled, count, clear


def round_e2m1(mag, unit):
    """mag / unit rounded to the eight levels; ties to the even code.  Both
    sides of each comparison are exact for 16-bit mag."""
    code = np.zeros(mag.shape, dtype=np.int64)
    for c, quarters in enumerate((1, 3, 5, 7, 10, 14, 20)):
        # between code c and c + 1: a tie stays at c when c is even
        past = 4 * mag > quarters * unit if c % 2 == 0 \
            else 4 * mag >= quarters * unit
        code = np.where(past, c + 1, code)
    return LEVELS[code]


def quantize_k(k, half: bool):
    """[..., D] -> the values that stand in the cache."""
    g = k.astype(np.float64).reshape(*k.shape[:-1], -1, 32)
    amax = np.abs(g).max(axis=-1, keepdims=True)
    finite = np.isfinite(amax)
    a = np.where(finite, amax, 1.0)
    e = np.full(a.shape, -126)
    for x in range(-125, 126):          # the least e with a <= 7 * 2^e
        e = np.where(a > 7 * 2.0 ** (x - 1), x, e)
    e = np.minimum(e, 13 if half else 125)
    unit = 2.0 ** e
    with np.errstate(invalid="ignore"):
        y = round_e2m1(np.abs(g), unit) * unit * np.sign(g)
    return np.where(finite, y, np.nan).reshape(k.shape)


def quantize_v(v):
    """[..., D] -> (values, scales): one scale for the D channels."""
    x = v.astype(np.float64)
    amax = np.abs(x).max(axis=-1, keepdims=True)
    finite = np.isfinite(amax)
    top = np.maximum(np.where(finite, amax, 1.0), 6 * 2.0 ** -100)
    with np.errstate(invalid="ignore"):
        y = round_e2m1(6 * np.abs(x), top) * (top / 6) * np.sign(x)
    return np.where(finite, y, np.nan), top / 6


def _attend_row(q, k, v, vscale, scale):
    """One query head's (result, bound) over the tokens of k, v and vscale."""
    kk, vv = k.astype(np.float64), v.astype(np.float64)
    qq = q.astype(np.float64)
    x = kk @ qq * scale
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.exp(x - x.max())
        w /= w.sum()
    # products are exact, sums of d + 1 terms are not, the score in base 2 and
    # log2 of the scale are rounded
    ls = np.abs(np.log2(vscale)) + 1
    ex = ((q.shape[-1] + 4) * 2.0 ** -24 * (np.abs(kk) @ np.abs(qq))
          * abs(scale) + (np.abs(x) * 2 + ls) * 2.0 ** -22).max()
    mass = w @ np.abs(vv)
    # float16 weights: 2^-11 relative (and as much again for approximations),
    # 2^-25 of the largest below its range
    return w @ vv, (mass * (2.0 ** -11 + 2.0 ** -14 + 3 * ex)
                    + 2.0 ** -25 * 6 * len(x) * vscale.max())


def attend(q, k, v, vscale, kv_len, q_len, scale=None):
    """q [B, T, Hq, D], k and v [B, L, H, D] as they stand in the cache, vscale
    [B, L, H, 1].  Returns (out, bound): how far a result computed with
    float16 weights, 32-bit sums and an unrounded output may be off."""
    b, t, hq, d = q.shape
    h = k.shape[2]
    g = hq // h
    scale = d ** -0.5 if scale is None else scale
    out = np.zeros(q.shape)
    bound = np.zeros(q.shape)
    for i in range(b):
        n, m = int(kv_len[i]), int(q_len[i])
        for j in range(min(m, t)):
            see = n - m + j + 1
            if see <= 0:
                continue
            for a in range(hq):
                out[i, j, a], bound[i, j, a] = _attend_row(
                    q[i, j, a], k[i, :see, a // g], v[i, :see, a // g],
                    vscale[i, :see, a // g, 0], scale)
    return out, bound


def ulp16(half: bool):
    """Largest relative rounding of the 16-bit type, and its smallest step."""
    return (2.0 ** -11, 2.0 ** -25) if half else (2.0 ** -8, 2.0 ** -134)


BLOCK = 32


def attend_blocks(q, selected, k, v, vscale, kv_len, q_len, scale=None):
    """As attend, over the positions of selected [B, T, H, N] blocks; those that
    name no block of k's length count as none, those named twice as one."""
    b, t, hq, d = q.shape
    n, h = k.shape[1:3]
    g = hq // h
    scale = d ** -0.5 if scale is None else scale
    out = np.zeros(q.shape)
    bound = np.zeros(q.shape)
    for i in range(b):
        for j in range(min(int(q_len[i]), t)):
            see = min(int(kv_len[i]) - int(q_len[i]) + j + 1, n)
            for a in range(hq):
                at = [p for x in sorted(set(selected[i, j, a // g].tolist()))
                      if x >= 0
                      for p in range(BLOCK * x, min(BLOCK * x + BLOCK, see))]
                if at:
                    out[i, j, a], bound[i, j, a] = _attend_row(
                        q[i, j, a], k[i, at, a // g], v[i, at, a // g],
                        vscale[i, at, a // g, 0], scale)
    return out, bound


def key_bounds(k):
    """[n <= 32, D] keys of a block -> (least, largest, unit) in whole units;
    unit 127 and zeros where there is a NaN."""
    d = k.shape[-1]
    if np.isnan(k).any():
        return np.zeros(d, int), np.zeros(d, int), 127
    top = np.abs(k).max()
    unit = -100
    if top > 0:
        unit = int(np.clip(np.frexp(top)[1] - 7, -100, 100))
    lo = np.floor(np.ldexp(k.min(axis=0), -unit))
    hi = np.ceil(np.ldexp(k.max(axis=0), -unit))
    return (np.clip(lo, -127, 127).astype(int),
            np.clip(hi, -127, 127).astype(int), unit)


def pack_query(q):
    """[G, D] query heads -> (P, N), whole numbers of 7 bits."""
    x = np.where(np.isfinite(q), q, 0.0).astype(np.float64)
    top = np.abs(x).max()
    if top == 0:
        z = np.zeros(q.shape[-1], int)
        return z, z
    z = np.rint(np.ldexp(x, 15 - int(np.frexp(top)[1]))).astype(np.int64)
    p, n = np.maximum(z, 0).sum(axis=0), np.maximum(-z, 0).sum(axis=0)
    shift = max(0, int(max(p.max(), n.max())).bit_length() - 7)
    return tuple(np.minimum((x + ((1 << shift) >> 1)) >> shift, 127)
                 for x in (p, n))


def select_blocks(q, bounds, kv_len, q_len, positions, blocks, first, recent):
    """q [B, T, Hq, D]; bounds[i][j][a]: key_bounds of row i's block j and KV head
    a, None where the table holds no page.  Python integers decide."""
    b, t, hq, _ = q.shape
    h = len(bounds[0][0]) if bounds and bounds[0] else 1
    g = hq // h
    out = np.full((b, t, h, blocks), -1, dtype=np.int32)
    for i in range(b):
        for j in range(min(int(q_len[i]), t)):
            see = min(int(kv_len[i]) - int(q_len[i]) + j + 1, positions)
            last = -(-see // BLOCK) - 1
            for a in range(h):
                p, n = pack_query(q[i, j, a * g:(a + 1) * g])
                ranked = []
                for x in range(last + 1):
                    if bounds[i][x][a] is None:
                        continue
                    lo, hi, unit = bounds[i][x][a]
                    if x < first or x > last - recent:
                        key = (2, 0)
                    elif unit == 127:
                        key = (1, 0)
                    else:   # in units of 2^-100
                        key = (0, int(p @ hi - n @ lo) << (unit + 100))
                    ranked.append((key, -x))
                ranked.sort(reverse=True)
                got = sorted(-x for _, x in ranked[:blocks])
                out[i, j, a, :len(got)] = got
    return out


def logprobs(logits, tokens, temperature=None, top=0):
    """(logprob, entropy, top tokens, top logprobs, and how far the first, the
    second and the last may be off computed in 32 bits)."""
    b, n, v = logits.shape
    lp, h = np.zeros((b, n)), np.zeros((b, n))
    ids = np.full((b, n, top), -1, dtype=np.int32)
    alt = np.full((b, n, top), -np.inf)
    tol = np.zeros((b, n)), np.zeros((b, n)), np.zeros((b, n, top))
    for i in range(b):
        t = 1.0 if temperature is None else float(temperature[i])
        for j in range(n):
            d = int(tokens[i, j])
            if not 0 <= d < v:
                continue
            x = logits[i, j].astype(np.float64)
            x = np.where(np.isnan(x), -np.inf, x)
            lp[i, j] = -np.inf
            order = np.argsort(-x, kind="stable")
            if x[order[0]] == -np.inf:
                continue
            if t > 0:
                with np.errstate(invalid="ignore", over="ignore"):
                    z = np.where(x == x[order[0]], 0.0, (x - x[order[0]]) / t)
            else:
                z = np.full(v, -np.inf)
                z[order[0]] = 0.0
            e = np.exp(z)
            rest = np.delete(e, order[0]).sum()
            log = np.log1p(rest)
            with np.errstate(invalid="ignore"):
                ze = np.where(e > 0, -z * e, 0.0)
                zze = np.where(e > 0, z * z * e, 0.0)
            lp[i, j] = z[d] - log
            h[i, j] = log + ze.sum() / (1 + rest)
            best = order[:top][x[order[:top]] > -np.inf]
            ids[i, j, :len(best)] = best
            alt[i, j, :len(best)] = z[best] - log
            if not t > 0:
                continue
            # the exponent is rounded four times, its power once more; a sum has
            # at most 64 additions behind one another; log1p and the result are
            # off by 2^-23 each
            u = 2.0 ** -24
            off = (u * (4 * ze.sum() + 4 * rest + 64 * rest) / (1 + rest)
                   + 4 * u * log)
            with np.errstate(invalid="ignore"):
                def of(y):
                    return np.where(y > -np.inf, off + 6 * u * np.abs(y), 0.0)
                tol[0][i, j] = of(z[d])
                tol[2][i, j, :len(best)] = of(z[best])
            tol[1][i, j] = (off + u * (4 * zze.sum() + 72 * ze.sum())
                            / (1 + rest) * (1 + rest / (1 + rest))
                            + off * ze.sum() / (1 + rest) + 4 * u * h[i, j])
    return lp, h, ids, alt, tol


class Pages:
    """A pool of pages by lists: free (its end on top), and each row's."""

    def __init__(self, num_pages, rows, width, page_size):
        self.free = list(range(num_pages - 1, -1, -1))
        self.rows = [[] for _ in range(rows)]
        self.width, self.page_size = width, page_size

    def resize(self, lengths):
        back = []
        for row, n in zip(self.rows, lengths):
            if n < 0:
                continue
            want = min(-(-int(n) // self.page_size), self.width)
            while len(row) < want and self.free:
                row.append(self.free.pop())
            back += row[want:]
            del row[want:]
        self.free += reversed(back)
        return [len(r) * self.page_size for r in self.rows[:len(lengths)]]

    def table(self):
        return np.array([r + [-1] * (self.width - len(r)) for r in self.rows],
                        dtype=np.int32)

    def slots(self, start, tokens, count=None):
        out = np.full((len(start), tokens), -1, dtype=np.int64)
        for r, s in enumerate(start):
            for i in range(tokens if count is None else min(tokens, count[r])):
                p = int(s) + i
                if 0 <= int(s) and p // self.page_size < len(self.rows[r]):
                    out[r, i] = (self.rows[r][p // self.page_size]
                                 * self.page_size + p % self.page_size)
        return out
