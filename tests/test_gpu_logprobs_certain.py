"""Log probabilities and entropies of rows with a token that is all but certain, relative to themselves: next to 1 a probability's logarithm is the sum of the others'.

Tolerances, in units u = 2^-24.  With r the sum of p = exp(-D) of all tokens but the likeliest, D = (largest - l) / T: an exponential's argument is off by 4 of itself
(difference, reciprocal of T, its product with log2(e), product), over all scalings to a new largest together too, and the exponential by 4 more.  A thread adds up 16 or 32 values,
17 additions at most, in one turn of at least 4096; a turn brings an addition, and where it has a new largest an exponential and a product, 7 together; lanes, warps and
blocks 22.  All of r has one sign, so that r is off by
    off(D) = 4 D + 4 + 17 + 7 (vocab / 4096 + 1) + 22
of itself, with D weighted as the terms of the sum are.  log(1 + r) is off by no more, relative to itself, and 2 for the answer's last steps; the log probability of another
token, - D - log(1 + r), by no more either.  Of the entropy, log(1 + r) + sum p D / (1 + r), the second sum has a difference and a product for each term, and 2 for each turn, besides, and is
divided by what r is off by.

Exponentials below 2^-126 count as nothing, as do those that a scaling below 2^-126 meets.  There are no more than vocab of them, each p below 2^-126: r and log(1 + r) are off by
vocab 2^-126 besides.  With p below 2^-126, D is above 126 ln 2 = 87.3, where p D falls as D grows: it is at most 88 2^-126, and the entropy is off by 89 times as much as r.
"""
from __future__ import annotations

import numpy as np
import pytest

from tests import f8_formulas as F
from tests.test_gpu_logprobs import rt, run  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def formula(logits, tokens, top, temperature):
    """(out, entropy, ids, best, D as weighted in r, as weighted in the entropy) in 64 bits; the likeliest token's own 1 is never added to."""
    n = len(logits)
    out, entropy, first, second = np.empty(n), np.empty(n), np.zeros(n), np.zeros(n)
    ids, best = np.full((n, top), -1), np.full((n, top), -np.inf)
    for row in range(n):
        x = logits[row].astype(np.float64)
        order = np.argsort(-x, kind="stable")
        order = order[x[order] > -np.inf]
        d = (x[order[0]] - x[order]) / np.float64(temperature[row])
        p = np.exp(-d[1:])
        r, weighted = p.sum(), (p * d[1:]).sum()
        log_sum = np.log1p(r)
        entropy[row] = log_sum + weighted / (1 + r)
        if weighted > 0:
            first[row], second[row] = weighted / r, (p * d[1:] ** 2).sum() / weighted
        at = np.flatnonzero(order == tokens[row])
        out[row] = -d[at[0]] - log_sum if len(at) else -np.inf
        k = min(top, len(order))
        ids[row, :k], best[row, :k] = order[:k], -d[:k] - log_sum
    return out, entropy, ids, best, first, second


def check(rt, logits, tokens, top=0, temperature=None, wide=False):
    n, vocab = logits.shape
    at = np.ones(n, np.float32) if temperature is None else np.asarray(temperature, np.float32)
    out, ent, ids, best = run(rt, logits, tokens, top, None if temperature is None else at)
    want_out, want_ent, want_ids, want_best, first, second = formula(logits, tokens, top, at)
    turns = 7 * (vocab / 4096 + 1)
    off = (4 * first + 4 + 17 + turns + 22) * F.U
    off_entropy = (4 * second + 6 + 17 + turns * 9 / 7 + 22) * F.U + off
    if wide:  # sums in 64 bits
        off, off_entropy = np.zeros(n), np.zeros(n)

    nothing = 0.0 if wide else vocab * 2.0**-126

    def near(got, want, off, least=nothing):
        some = want > -np.inf
        assert np.array_equal(got > -np.inf, some)
        miss = np.abs(got[some].astype(np.float64) - want[some]) - (off[some] + 2 * F.U) * np.abs(want[some]) - least
        assert (miss <= 0).all(), (miss.max(), got[some][miss.argmax()], want[some][miss.argmax()])

    assert np.array_equal(ids, want_ids)
    near(out, want_out, off)
    near(ent, want_ent, np.maximum(off, off_entropy), 89 * nothing)
    near(best, want_best, np.repeat(off[:, None], top, 1))


MARGINS = (3, 5, 8, 10, 12, 16, 17, 20, 25, 30, 40)


def two_tokens(kind, vocab):
    """Rows of two tokens, at each margin, the two in one vector, thread, warp, block of threads, and in different ones."""
    each = 16 // np.dtype(kind).itemsize
    rng = np.random.default_rng(vocab)
    rows, tokens = [], []
    for margin in MARGINS:
        for apart in (1, each, 31 * each, 256 * each, 512 * each, 1024 * each, 2048 * each, vocab // 2):
            first = int(rng.integers(0, vocab))
            other = (first + apart) % vocab
            row = np.full(vocab, -np.inf, kind)
            row[first] = rng.uniform(-3, 12)
            row[other] = row[first] - kind(margin)
            rows.append(row)
            tokens.append(first if rng.random() < 0.8 else other)
    return np.array(rows), np.array(tokens)


@pytest.mark.parametrize("kind", [np.float32, np.float16])
@pytest.mark.parametrize("vocab", [900, 7001, 32003, 70000])
@pytest.mark.parametrize("n", [1, 20, 352])
def test_two_tokens(rt, kind, vocab, n):  # noqa: F811
    logits, tokens = two_tokens(kind, vocab)
    if n > len(logits):
        logits, tokens = np.tile(logits, (n // len(logits), 1)), np.tile(tokens, n // len(tokens))
    rng = np.random.default_rng(n)
    temperature = rng.uniform(0.5, 1.2, len(logits))
    step = n if n > 1 else 3
    for r in range(0, len(logits) - min(n, 20) + 1, step):
        check(rt, logits[r:r + n], tokens[r:r + n])
        check(rt, logits[r:r + n], tokens[r:r + n], 3, temperature[r:r + n])


@pytest.mark.parametrize("kind", [np.float32, np.float16])
@pytest.mark.parametrize("n", [1, 20, 330])
def test_one_token_above_all_others(rt, kind, n):  # noqa: F811
    rng = np.random.default_rng(n)
    vocab = 20011
    logits = (rng.standard_normal((max(n, len(MARGINS)), vocab)) * 0.7).astype(kind)
    tokens = rng.integers(0, vocab, len(logits))
    logits[np.arange(len(logits)), tokens] = [12 + MARGINS[r % len(MARGINS)] for r in range(len(logits))]
    for r in range(0, len(logits) - n + 1, n):
        check(rt, logits[r:r + n], tokens[r:r + n], 1)
        check(rt, logits[r:r + n], tokens[r:r + n], 20, rng.uniform(0.5, 1.2, n))


@pytest.mark.parametrize("n", [1, 300])
def test_the_same_row_whatever_else_is_in_the_call(rt, n):  # noqa: F811
    """A row's answers do not depend on the number of rows beyond what its sums are off by; equal largest ones are as likely as each other."""
    vocab = 30011
    rng = np.random.default_rng(6)
    x = (rng.standard_normal((4, vocab)) * 3).astype(np.float32)
    x[0, 17], x[1, [5, 6]], x[2, [9, 20000]] = 30, 40, 25
    x[3] = 0.25
    logits = np.tile(x, (n, 1))[:max(n, 4)]
    for r in range(0, len(logits) - n + 1, n):
        check(rt, logits[r:r + n], np.resize([17, 6, 9, 3], len(logits))[r:r + n], 2)


@pytest.mark.parametrize("n", [1, 300])
def test_rows_that_are_summed_in_64_bits(rt, n):  # noqa: F811
    vocab = 9001
    for top, step, at in ((0.0, -2e-30, 1e-31), (3e30, -3e24, 1.4e23), (-2e30, -1e25, 4e23)):
        x = np.full((n, vocab), -np.inf, np.float32)
        x[:, 77], x[:, 78], x[:, 5000] = top, np.float32(top + step), np.float32(top + 2 * step)
        check(rt, x, [77] * n, 3, [at] * n, wide=True)
        check(rt, x, [78] * n, 1, [at] * n, wide=True)
