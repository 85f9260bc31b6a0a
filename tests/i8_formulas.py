"""The formulas of the 8-bit integer passes and of the verification of drafted tokens in 64 bits, in numpy."""
from __future__ import annotations

import numpy as np

HALF_STEP = {np.float32: 2.0**-24, np.float16: 2.0**-11}


def pitch(cols: int) -> int:
    return (cols + 15) // 16 * 16


def rows_i8(x, *, x2=None, residual=None, norm=None, eps=1e-6):
    """(q, scale, sum) of activation rows x [ntok][cols]."""
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
        scale = (np.abs(v).max(1) / 127.0).astype(np.float32)
        scale[~np.isfinite(v).all(1) | ~np.isfinite(scale)] = np.nan
        q = np.where(scale[:, None] > 0, np.rint(v / scale[:, None].astype(np.float64)), 0.0)
        q = np.where(np.isnan(scale)[:, None], 0.0, np.clip(q, -127, 127))
    return q.astype(np.int8), scale, total


def qmm_i8(w, w_scale, q, q_scale):
    """(y in 64 bits, the sums themselves)."""
    sums = q.astype(np.int64) @ w.astype(np.int64).T if q.shape[1] < 4096 else np.rint(q.astype(np.float64) @ w.astype(np.float64).T).astype(np.int64)
    return sums * q_scale.astype(np.float64)[:, None] * w_scale.astype(np.float64), sums


def spread(logits, temperature):
    """A row's probabilities."""
    x = logits.astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    w = np.zeros_like(x)
    top = x.max()
    if top == -np.inf:
        return w
    if not temperature > 0:
        w[int(np.argmax(x))] = 1.0
        return w
    with np.errstate(all="ignore"):
        some = x > -np.inf
        w[some] = np.where(x[some] == top, 1.0, np.exp((x[some] - top) / np.float64(temperature)))
        if temperature == np.inf:
            w[some] = np.where((x[some] == top) | np.isfinite(top), 1.0, 0.0)
    return w / w.sum()


def verify(target, draft, tokens, uniforms, lens=None, temperature=None):
    """out [seqs][drafts + 2] of Runtime.verify."""
    n, rows, vocab = target.shape
    k = rows - 1
    out = np.full((n, k + 2), -1, np.int32)
    for s in range(n):
        at = 1.0 if temperature is None else temperature[s]
        drafts = k if lens is None else min(k, max(0, int(lens[s])))
        j, rest = 0, None
        while j < drafts:
            p, token = spread(target[s, j], at), int(tokens[s, j])
            inside = 0 <= token < vocab
            if draft is not None:
                q = spread(draft[s, j], at)
            else:
                q = np.zeros(vocab)
                if inside:
                    q[token] = 1.0
            if not inside or not float(uniforms[s, j]) * q[token] < p[token]:
                rest = np.maximum(p - q, 0.0)
                if not rest.sum() > 0:
                    rest = p
                break
            out[s, 1 + j] = token
            j += 1
        if rest is None:
            rest = spread(target[s, j], at)
        out[s, 0] = j
        sums = np.cumsum(rest)
        if sums[-1] > 0:
            above = np.nonzero((sums > float(uniforms[s, k]) * sums[-1]) & (rest > 0))[0]
            out[s, 1 + j] = above[0] if len(above) else np.nonzero(rest > 0)[0][-1]
    return out
