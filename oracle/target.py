"""The operators on the target model's side of a step, by their definitions, in
numpy and 64 bits: verification of drafts, the rounding of keys and values to
4 bits, and attention over what they then stand for."""

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
                kk = k[i, :see, a // g].astype(np.float64)
                vv = v[i, :see, a // g].astype(np.float64)
                qq = q[i, j, a].astype(np.float64)
                x = kk @ qq * scale
                with np.errstate(invalid="ignore", over="ignore"):
                    w = np.exp(x - x.max())
                    w /= w.sum()
                out[i, j, a] = w @ vv
                # products are exact, sums of d + 1 terms are not, the score
                # in base 2 and log2 of the scale are rounded
                ls = np.abs(np.log2(vscale[i, :see, a // g, 0])) + 1
                ex = ((d + 4) * 2.0 ** -24 * (np.abs(kk) @ np.abs(qq))
                      * abs(scale) + (np.abs(x) * 2 + ls) * 2.0 ** -22).max()
                mass = w @ np.abs(vv)
                # float16 weights: 2^-11 relative (and as much again for
                # approximations), 2^-25 of the largest below its range
                bound[i, j, a] = (mass * (2.0 ** -11 + 2.0 ** -14 + 3 * ex)
                                  + 2.0 ** -25 * 6 * see
                                  * vscale[i, :see, a // g].max())
    return out, bound


def ulp16(half: bool):
    """Largest relative rounding of the 16-bit type, and its smallest step."""
    return (2.0 ** -11, 2.0 ** -25) if half else (2.0 ** -8, 2.0 ** -134)


