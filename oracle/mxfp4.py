"""MXFP4 pools, attention weights and eviction in plain NumPy and 64 bits (the oracle of their tests).

Blocks of 32 elements: E2M1 codes (OCP Microscaling Formats v1.0, section 5.3.3) and an E8M0 scale
(section 5.4.1), chosen by its section 6.3: the largest magnitude's exponent less E2M1's largest, 2.
"""
import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
NONE = 0xFFFFFFFF


def quantise(x):
    """x: [..., d] floats.  Codes [..., d / 2] and scales [..., d / 32], uint8."""
    b = np.asarray(x, np.float64).reshape(*np.shape(x)[:-1], -1, 32)
    top = np.abs(b).max(-1, keepdims=True)
    bad = ~np.isfinite(b).all(-1, keepdims=True)
    none = bad | (top == 0)
    exponent = np.where(none, -125, np.frexp(np.where(none, 1.0, top))[1] - 1)
    s = np.clip(exponent + 127 - 2, 0, 254).astype(np.int64)
    y = np.where(bad, 0.0, b) / 2.0 ** (s.astype(np.float64) - 127)
    far = np.abs(np.abs(y)[..., None] - LEVELS)
    code = far.argmin(-1)                                   # the lower of two equally near
    up = np.minimum(code + 1, 7)
    tie = (np.take_along_axis(far, code[..., None], -1) == np.take_along_axis(far, up[..., None], -1))[..., 0]
    code = np.where(tie & (code % 2 == 1), up, code)        # ... unless it is odd
    code = (code + 8 * np.signbit(y)).astype(np.uint8)
    code = np.where(bad, 0, code).astype(np.uint8).reshape(*np.shape(x)[:-1], -1, 2)
    return code[..., 0] | code[..., 1] << 4, np.where(bad, 255, s)[..., 0].astype(np.uint8)


def dequantise(codes, scales):
    """Values [..., d] in 64 bits."""
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    x = LEVELS[c & 7] * np.where(c & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return (x.reshape(*x.shape[:-1], -1, 32) * s[..., None]).reshape(x.shape)


def keys_of(plane, table, n, page):
    """[kv head, key, d] of one sequence from a plane of values [page][kv head][page_size][d].  Table entries
    outside the plane read as zeros."""
    rows = []
    for i in range(-(-n // page)):
        e = int(table[i])
        rows.append(plane[e] if e < len(plane) else np.zeros_like(plane[0]))
    return np.concatenate(rows, 1)[:, :n]


def softmax_weights(q, k, first, scale):
    """q: [rows, hq, d], k: [hkv, keys, d]; row r attends keys <= first + r.  [hkv, rows, group, keys]."""
    rows, hq, d = q.shape
    hkv, keys, _ = k.shape
    x = q.reshape(rows, hkv, hq // hkv, d)
    s = np.einsum("rhgd,hkd->hrgk", x.astype(np.float64), np.nan_to_num(k)) * scale
    s = np.where(np.isnan(k).any(-1)[:, None, None, :], np.nan, s)
    hidden = np.arange(keys)[None, :] > first + np.arange(rows)[:, None]
    s = np.where(hidden[None, :, None, :], -np.inf, s)
    with np.errstate(invalid="ignore"):
        p = np.exp(s - s.max(-1, keepdims=True))
    return p / p.sum(-1, keepdims=True)


def attention(q, k, v, first, scale):
    """[rows, hq, d]; NaN values reach the rows that attend their key alone."""
    p = softmax_weights(q, k, first, scale)
    hkv, rows, group, keys = p.shape
    bad = np.isnan(v)
    o = np.einsum("hrgk,hkd->rhgd", p, np.where(bad, 0.0, v))
    live = np.arange(keys)[None, :] <= first + np.arange(rows)[:, None]
    hit = np.einsum("rk,hkd->rhd", live.astype(np.float64), bad.astype(np.float64)) > 0
    o = np.where(hit[:, :, None, :], np.nan, o)
    return o.reshape(rows, hkv * group, -1)


def order(mass):
    """Whole numbers in the floats' IEEE total order."""
    b = np.asarray(mass, np.float32).view(np.int32).astype(np.int64)
    return np.where(b < 0, -1 - (b & 0x7FFFFFFF), b)


def select(mass, budget, recent):
    """mass: [n] of one sequence and KV head.  The kept keys, ascending: the last min(recent, budget) and the
    heaviest of the others, ties to the lower index."""
    n = len(mass)
    if n <= budget:
        return np.arange(n)
    r = min(recent, budget)
    key = order(mass[:n - r])
    best = np.lexsort((np.arange(n - r), -key))[:budget - r]
    return np.sort(np.concatenate([best, np.arange(n - r, n)]))
