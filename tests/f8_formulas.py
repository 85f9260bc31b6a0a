"""The formulas of the passes in 8-bit floating point and of log probabilities in 64 bits, in numpy."""
from __future__ import annotations

import numpy as np

BLOCK = 128
MOST = 448.0
U = 2.0**-24  # half a step of fp32, relative


def _codes():
    """The value of each of the 256 e4m3 bytes."""
    b = np.arange(256)
    exponent, mantissa = (b >> 3) & 15, b & 7
    v = np.where(exponent == 0, mantissa / 8 * 2.0**-6, (1 + mantissa / 8) * 2.0 ** (exponent - 7.0))
    v[(b & 127) == 127] = np.nan
    return np.where(b & 128, -v, v)


CODES = _codes()
_POSITIVE = CODES[:127]  # 0 to 448, in order


def encode(t):
    """The nearest e4m3 byte, ties to the even one, beyond 448 that; t is fp32 or wider."""
    t = np.asarray(t, np.float64)
    a = np.minimum(np.abs(t), MOST)
    above = np.searchsorted(_POSITIVE, a)  # the first that is no less
    below = np.maximum(above - 1, 0)
    low, high = a - _POSITIVE[below], _POSITIVE[above] - a
    code = np.where((low < high) | ((low == high) & (below % 2 == 0)), below, above)
    return (code | np.where(np.signbit(t), 128, 0)).astype(np.uint8)


def step(t):
    """How far e4m3 values are apart at t."""
    e = np.floor(np.log2(np.maximum(np.abs(np.asarray(t, np.float64)), 2.0**-6)))
    return 2.0 ** (np.minimum(e, 8) - 3)


def pitch(cols):
    return (cols + 15) // 16 * 16


def blocks(n):
    return (n + BLOCK - 1) // BLOCK


def scale_pitch(ntok):
    return (ntok + 3) // 4 * 4


def values(x, *, x2=None, residual=None, norm=None, eps=1e-6):
    """(n in 64 bits, sum) of activation rows x [ntok][cols]."""
    total = None
    with np.errstate(all="ignore"):
        v = x.astype(np.float64)
        if x2 is not None:
            v = v / (1.0 + np.exp(-v)) * x2.astype(np.float64)
        if residual is not None:
            total = (x.astype(np.float32) + residual.astype(np.float32)).astype(x.dtype)
            v = total.astype(np.float64)
        if norm is not None:
            v = v / np.sqrt((v * v).mean(1, keepdims=True) + np.float64(np.float32(eps))) * norm.astype(np.float64)
    return v, total


def scales_of(n):
    """max |n| / 448 of each block of columns, [blocks][ntok], in 64 bits; NaN where one of them is not finite."""
    ntok, cols = n.shape
    out = np.empty((blocks(cols), ntok))
    for b in range(blocks(cols)):
        part = n[:, b * BLOCK:(b + 1) * BLOCK]
        out[b] = np.where(np.isfinite(part).all(1), np.abs(part).max(1), np.nan) / MOST
    return out


def spread_scales(s, cols):
    """[blocks][ntok] -> [ntok][cols]"""
    return np.repeat(s.T, BLOCK, 1)[:, :cols]


def qmm(w, w_scale, q, q_scale):
    """(y in 64 bits, the same of the absolute values) of bytes w [rows][cols], q [ntok][cols]; w_scale [blocks(rows)][blocks(cols)], q_scale [blocks(cols)][ntok]."""
    rows, cols = w.shape
    x = CODES[q] * spread_scales(q_scale.astype(np.float64), cols)
    v = CODES[w] * np.repeat(np.repeat(w_scale.astype(np.float64), BLOCK, 0)[:rows], BLOCK, 1)[:, :cols]
    return x @ v.T, np.abs(x) @ np.abs(v).T


def less(logits, temperature):
    """(logit - largest) / T of a row in 64 bits, -inf where p is nothing; and the places in order of preference, those that are not masked."""
    x = logits.astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    d = np.full(len(x), -np.inf)
    if len(order) == 0:
        return d, order
    top = x[order[0]]
    some = x > -np.inf
    if not temperature > 0:
        d[order[0]] = 0.0
    elif top == np.inf:
        d[x == top] = 0.0
    elif temperature > 1e30:
        d[some] = 0.0
    else:
        with np.errstate(all="ignore"):
            d[some] = (x[some] - top) / np.float64(temperature)
    return d, order


def logprobs(logits, tokens, top=0, temperature=None):
    """(out, entropy, top_ids, top_out) in 64 bits."""
    n, vocab = logits.shape
    out, entropy = np.full(n, -np.inf), np.zeros(n)
    ids, best = np.full((n, top), -1, np.int32), np.full((n, top), -np.inf)
    for r in range(n):
        d, order = less(logits[r], 1.0 if temperature is None else temperature[r])
        if len(order) == 0:
            continue
        e = np.exp(d)
        log_sum = np.log(e.sum())
        entropy[r] = log_sum - (e[e > 0] * d[e > 0]).sum() / e.sum()
        if 0 <= tokens[r] < vocab:
            out[r] = d[tokens[r]] - log_sum
        k = min(top, len(order))
        ids[r, :k] = order[:k]
        best[r, :k] = d[order[:k]] - log_sum
    return out, entropy, ids, best
