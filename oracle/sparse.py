"""Rotation from given frequencies, page summaries, page selection and attention over selected pages in plain NumPy and
64 bits (the oracle of their tests)."""
import math

import numpy as np

from oracle import mxfp4 as M

NONE = 0xFFFFFFFF


# ------------------------------------------------------------------ rotation

def rotated(x, table, interleaved):
    """Heads [rows, heads, d] with the pairs of table [rows, pairs, 2] rotated, and the sum of each element's two
    products' magnitudes (of the others their own)."""
    x, table = np.asarray(x, np.float64), np.asarray(table, np.float64)
    out, size = x.copy(), np.abs(x)
    pairs = table.shape[1]
    for i in range(pairs):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
        c, s = table[:, None, i, 0], table[:, None, i, 1]
        out[..., a] = x[..., a] * c - x[..., b] * s
        out[..., b] = x[..., b] * c + x[..., a] * s
        size[..., a] = np.abs(x[..., a] * c) + np.abs(x[..., b] * s)
        size[..., b] = np.abs(x[..., b] * c) + np.abs(x[..., a] * s)
    return out, size


def normalised(x, weight, eps):
    x = np.asarray(x, np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)


# ------------------------------------------------------------------ pages

def codes(x):
    """Whole numbers within +-127 and the power of two that they count, for the last axis of finite values."""
    x = np.asarray(x, np.float64)
    top = np.abs(x).max(-1, keepdims=True)
    exponent = np.where(top == 0, -126, np.frexp(np.where(top == 0, 1.0, top))[1] - 1 - 6)
    unit = 2.0 ** np.maximum(exponent, -126)
    return np.clip(np.rint(x / unit), -127, 127).astype(np.int64), unit[..., 0]


def summary(keys):
    """keys: [heads, tokens, d] of one full page.  codes [heads, 2, d], scales [heads]."""
    keys = np.asarray(keys, np.float64)
    bad = ~np.isfinite(keys).all((1, 2))
    keys = np.where(bad[:, None, None], 0.0, keys)
    c, unit = codes(np.concatenate([keys.max(1), keys.min(1)], -1))
    return (np.where(bad[:, None, None], 0, c.reshape(len(keys), 2, -1)).astype(np.int8),
            np.where(bad, np.inf, unit).astype(np.float32))


def scores(q, page_codes, page_scales):
    """q: [group, d] of one row and KV head; page_codes [pages, 2, d], page_scales [pages].  Scores [pages] in f32."""
    c, unit = codes(q)
    sums = np.maximum(c, 0) @ page_codes[:, 0].astype(np.int64).T + np.minimum(c, 0) @ page_codes[:, 1].astype(np.int64).T
    with np.errstate(invalid="ignore"):
        s = (sums.astype(np.float32) * unit.astype(np.float32)[:, None]) * page_scales[None].astype(np.float32)
    s = np.where(np.isinf(page_scales)[None], np.float32(np.inf), s)
    return s.max(0) + np.float32(0)


def select(score, n, budget, first, recent):
    """The pages that stay of n, ascending; score [n]."""
    if n <= budget:
        return np.arange(n)
    middle = np.arange(first, n - recent)
    best = middle[np.lexsort((middle, -M.order(score[middle])))[:budget - first - recent]]
    return np.concatenate([np.arange(first), np.sort(best), np.arange(n - recent, n)])


def attention(q, k, v, pages, count, position, page, scale):
    """One row and KV head: q [group, d], k and v [pool pages + 1, page, d] values of the table's entries (the last one:
    zeros, outside the pool), pages: [(logical page, entry)].  (out [group, d], sum of the weights' magnitudes times V's)."""
    ks, vs = [], []
    for sel, entry in pages[:count]:
        live = min(page, position + 1 - sel * page)
        if live > 0:
            ks.append(k[entry][:live])
            vs.append(v[entry][:live])
    if not ks:
        return np.zeros(q.shape), np.zeros(q.shape)
    ks, vs = np.concatenate(ks).astype(np.float64), np.concatenate(vs).astype(np.float64)
    s = np.asarray(q, np.float64) @ ks.T * scale
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    return p @ vs, p @ np.abs(vs)


# ------------------------------------------------------------------ frequencies

def frequencies(n, base, scaling=None, factor=1.0, context=0.0, low=1.0, high=32.0):
    if scaling == "base":
        base = base * factor ** (n / (n - 2))
    out = []
    for i in range(n // 2):
        f = base ** (-2 * i / n)
        if scaling == "linear":
            f /= factor
        elif scaling in ("turns", "index"):
            if scaling == "turns":
                keep = (context * f / (2 * math.pi) - low) / (high - low)
            else:
                at = lambda turns: n / 2 * math.log(context / (2 * math.pi * turns)) / math.log(base)  # noqa: E731
                a, b = max(math.floor(at(high)), 0), min(math.ceil(at(low)), n - 1)
                keep = 1 - (i - a) / (b - a if b > a else 0.001)
                if context / (2 * math.pi) <= low:  # even the first pair's turns
                    keep = 0.0
            keep = min(max(keep, 0.0), 1.0)
            f = f * keep + f / factor * (1 - keep)
        out.append(f)
    return np.array(out)
