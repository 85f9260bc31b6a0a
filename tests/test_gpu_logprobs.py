"""Log probabilities on the GPU against their definition in 64 bits (tests/f8_formulas.py).  Places are whole numbers: they are equal.

Tolerances, in units u = 2^-24.  With S the sum of e = exp((l - m) / T): the argument d / T of an exponential is off by 4 of itself (difference, reciprocal of T, its
product with log2(e), product) and the exponential by 4 more; weighted by p, |d| / T comes to the entropy H at most.  A lane adds up 8192 / 512 values of fp32 (16-bit ones: twice
as many, in two sums) in 16 additions, and those sums one after the other: for each an addition, and where it brings a new largest an exponential and a product, 7 together for at
most vocab / 8192 + 1 of them.  Lanes, warps and blocks take two such scalings and 10 additions more, 22.  So S, and log S, is off by
    sums = (4 H + 4 + 16 + 7 (vocab / 8192 + 1) + 22) u,
a log probability by that and 3 of itself, and the entropy, log S + U / S, by sums (1 + 3 H).
"""
from __future__ import annotations

import numpy as np
import pytest

from tests import f8_formulas as F
from tests.test_gpu_verify_status import late  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    from vinf_3080ti_b200.runtime import Runtime

    r = Runtime()
    yield r
    r.synchronize()
    r.close()


def put(rt, name, a):
    a = np.ascontiguousarray(a)
    rt.alloc(name, a.size, a.dtype.itemsize)
    rt.write(name, a)


def run(rt, logits, tokens, top=0, temperature=None, entropy=True, top_out=True):
    n, vocab = logits.shape
    put(rt, "logits", logits)
    put(rt, "tokens", np.asarray(tokens, np.int32))
    if temperature is not None:
        put(rt, "temp", np.asarray(temperature, np.float32))
    for name, count in (("out", n), ("entropy", n), ("best", n * top)):
        put(rt, name, np.full(count + 3, 7.0, np.float32))
    put(rt, "ids", np.full(n * top + 3, 555, np.int32))
    rt.logprobs("logits", "tokens", vocab, n, out="out", entropy="entropy" if entropy else None, top=top, top_ids="ids" if top else None,
                top_out="best" if top and top_out else None, temperature=None if temperature is None else "temp")
    rt.synchronize()
    out, ent, best = (rt.read_array(name) for name in ("out", "entropy", "best"))
    ids = np.frombuffer(rt.read("ids"), np.int32)
    assert (out[n:] == 7).all() and (ent[n if entropy else 0:] == 7).all() and (best[n * top if top_out else 0:] == 7).all() and (ids[n * top:] == 555).all()
    return out[:n], ent[:n] if entropy else None, ids[:n * top].reshape(n, top), best[:n * top].reshape(n, top) if top_out else None


def check(rt, logits, tokens, top=0, temperature=None, **kw):
    at = None if temperature is None else np.asarray(temperature, np.float32)
    out, ent, ids, best = run(rt, logits, tokens, top, at, **kw)
    want_out, want_ent, want_ids, want_best = F.logprobs(logits, tokens, top, at)
    assert np.array_equal(ids, want_ids), np.argwhere(ids != want_ids)[:5]
    sums = (4 * want_ent + 4 + 16 + 7 * (logits.shape[1] / 8192 + 1) + 22) * F.U

    def near(got, want, off):
        # answers are fp32: what is a half step or more beyond its largest, 2^128 - 2^104, is infinite there
        want = np.where(want <= -(2.0**128 - 2.0**103), -np.inf, want)
        fine = np.isfinite(want)
        assert np.array_equal(got[~fine], want[~fine].astype(np.float32)), (got[~fine][:5], want[~fine][:5])
        miss = np.abs(got[fine] - want[fine]) - off[fine]
        assert (miss <= 0).all(), (miss.max(), got[fine][miss.argmax()], want[fine][miss.argmax()])

    near(out, want_out, sums + 3 * F.U * np.abs(np.where(np.isfinite(want_out), want_out, 0)))
    if ent is not None:
        near(ent, want_ent, sums * (1 + 3 * want_ent))
    if best is not None and top:
        near(best, want_best, sums[:, None] + 3 * F.U * np.abs(np.where(np.isfinite(want_best), want_best, 0)))
    return out, ent, ids, best


VOCABS = [1, 2, 3, 7, 8, 31, 32, 33, 100, 511, 512, 513, 1000, 4095, 4096, 4097, 8191, 8193, 20000, 32003, 151936]


@pytest.mark.parametrize("kind", [np.float32, np.float16])
@pytest.mark.parametrize("vocab", VOCABS)
def test_every_vocabulary(rt, vocab, kind):
    rng = np.random.default_rng(vocab)
    for n in (1, 2, 5):
        logits = (rng.standard_normal((n, vocab)) * 3).astype(kind)
        tokens = rng.integers(0, vocab, n)
        check(rt, logits, tokens)
        check(rt, logits, tokens, top=20)
        check(rt, logits, tokens, top=1, temperature=rng.uniform(0.3, 2, n))
        check(rt, logits, logits.argmax(1), top=32, entropy=False)


@pytest.mark.parametrize("n", [8, 9, 13, 18, 19, 37, 64, 74, 75, 100, 148, 149, 200, 296, 297, 700])
def test_every_number_of_rows(rt, n):
    rng = np.random.default_rng(n)
    for vocab, kind in ((20011, np.float32), (30000, np.float16), (777, np.float32)):
        logits = (rng.standard_normal((n, vocab)) * 2).astype(kind)
        check(rt, logits, rng.integers(0, vocab, n), top=int(rng.integers(0, 33)), temperature=rng.uniform(0.5, 1.5, n))


@pytest.mark.parametrize("n", [1, 5, 40, 300])
def test_ties_go_to_the_lowest_place(rt, n):
    """Rows of few values, of one value, of two halves: more candidates than any list holds."""
    rng = np.random.default_rng(n)
    vocab = 30011
    few = rng.integers(0, 4, (n, vocab)).astype(np.float32)
    check(rt, few, rng.integers(0, vocab, n), top=32)
    same = np.full((n, vocab), -2.5, np.float32)
    check(rt, same, rng.integers(0, vocab, n), top=32)
    same[:, vocab // 2:] = 1.5
    check(rt, same.astype(np.float16), rng.integers(0, vocab, n), top=7)
    zeros = np.where(rng.integers(0, 2, (n, vocab)) == 0, np.float32(0.0), np.float32(-0.0))
    check(rt, zeros, rng.integers(0, vocab, n), top=20)


@pytest.mark.parametrize("n", [1, 5, 300])
def test_sorted_rows(rt, n):
    """The largest last, or first: every part of a row has another's largest beside it."""
    vocab = 20000
    up = np.tile(np.linspace(-10, 10, vocab, dtype=np.float32), (n, 1))
    check(rt, up, [vocab - 1] * n, top=32)
    check(rt, np.ascontiguousarray(up[:, ::-1]), [0] * n, top=32)
    saw = np.tile((np.arange(vocab) % 512).astype(np.float32) / 100, (n, 1))
    check(rt, saw, [511] * n, top=32)


@pytest.mark.parametrize("kind", [np.float32, np.float16])
@pytest.mark.parametrize("vocab", [40, 5003, 70000])
def test_masked_rows(rt, vocab, kind):
    """Rows of which a few logits are left, or one, or none; masked by -inf, by NaN, by the type's lowest value."""
    rng = np.random.default_rng(vocab)
    for fill in (-np.inf, np.nan, np.finfo(kind).min):
        logits = (rng.standard_normal((7, vocab)) * 3).astype(kind)
        for r, left in enumerate((0, 1, 2, 5, 19, 21, 30)):
            keep = rng.choice(vocab, left, replace=False)
            row = np.full(vocab, fill, kind)
            row[keep] = logits[r, keep]
            logits[r] = row
        tokens = [0, int(np.nanargmax(logits[1])), 3, vocab - 1, -1, vocab, 2**31 - 1]
        for top in (0, 1, 20, 32):
            check(rt, logits, tokens, top=top)
            check(rt, logits, tokens, top=top, temperature=[0.5, 0.0, 2.0, -1.0, np.nan, 1e31, 1e-3])


def test_infinite_logits_and_extreme_values(rt):
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((12, 5000)) * 3).astype(np.float32)
    x[0, [7, 4000]] = np.inf
    x[1, 5] = np.inf
    x[2] *= 1e30
    x[3] *= 1e36
    x[4] = -3e38
    x[4, 77] = -2e38
    x[5] = np.finfo(np.float32).max
    x[6, 3] = 3e38
    x[7, 3], x[7, 4] = -3e38, 1e3
    x[8] *= 1e-38
    x[9] += 1e6
    x[10] = -1e5
    x[11, ::2], x[11, 1::2] = 3.4e38, -3.4e38
    for at in (None, [1.0] * 12, [1e-3] * 12, [1e29] * 12, [1e38] * 12, [0.0] * 12, [1e-38] * 12, [1e-44] * 12):
        check(rt, x, [7, 4, 100, 5, 77, 0, 3, 3, 9, 10, 4999, 1], top=8, temperature=at)


def test_a_token_that_is_all_but_certain(rt):
    """Its log probability is next to zero, the others' far below; a margin at every size."""
    rng = np.random.default_rng(4)
    x = rng.standard_normal((9, 50000)).astype(np.float32)
    for r, margin in enumerate((5, 10, 12, 15, 20, 25, 30, 60, 110)):
        x[r, 123] = margin
    out, ent, _, _ = check(rt, x, [123] * 9, top=3)
    check(rt, x, [124] * 9, top=3)
    assert (out <= 0).all() and (ent >= 0).all()


@pytest.mark.parametrize("kind", [np.float32, np.float16])
def test_rows_that_begin_anywhere(rt, kind):
    """A vocabulary that is odd: every row lies on the grid of 16 bytes in another way; and a buffer that is longer than what is asked for."""
    rng = np.random.default_rng(5)
    for vocab in (4001, 4002, 4003, 4005, 4007):
        x = (rng.standard_normal((17, vocab)) * 3).astype(kind)
        put(rt, "logits", np.concatenate([x.reshape(-1), np.full(100, np.inf, kind)]))
        check(rt, x, rng.integers(0, vocab, 17), top=5)


@pytest.mark.parametrize("seqs", [1, 20, 300])
def test_captured_and_replayed(rt, seqs):
    rng = np.random.default_rng(seqs)
    vocab = 9001
    x = rng.standard_normal((3, seqs, vocab)).astype(np.float32) * 3
    tokens = rng.integers(0, vocab, seqs).astype(np.int32)
    eager = [run(rt, x[i], tokens, top=5) for i in range(3)]
    rt.capture_begin()
    rt.logprobs("logits", "tokens", vocab, seqs, out="out", entropy="entropy", top=5, top_ids="ids", top_out="best")
    graph = rt.capture_end()
    for i in range(3):
        rt.write("logits", x[i])
        rt.graph_launch(graph)
        rt.synchronize()
        assert np.array_equal(rt.read_array("out")[:seqs], eager[i][0]) and np.array_equal(rt.read_array("entropy")[:seqs], eager[i][1])
        assert np.array_equal(np.frombuffer(rt.read("ids"), np.int32)[:seqs * 5].reshape(seqs, 5), eager[i][2])
        assert np.array_equal(rt.read_array("best")[:seqs * 5].reshape(seqs, 5), eager[i][3])
    rt.graph_destroy(graph)


def test_answers_from_logits_that_a_failed_launch_has_left(late):
    """Undefined until the failure has been reported; captured ones too."""
    rt, run_out = late
    put(rt, "t", np.zeros(2, np.int32))
    for name in ("o", "e", "v"):
        rt.alloc(name, 6)
    put(rt, "i", np.zeros(6, np.int32))

    def call():
        rt.logprobs("target", "t", 64, 2, out="o", entropy="e", top=3, top_ids="i", top_out="v")

    def answers():
        return [rt.read(name) for name in ("o", "e", "i", "v")]

    call()
    want = answers()
    rt.capture_begin()
    call()
    graph = rt.capture_end()
    for again in (call, lambda: rt.graph_launch(graph)):
        run_out()
        again()
        o, e, i, v = answers()
        assert np.isnan(np.frombuffer(o, np.float32)[:2]).all() and np.isnan(np.frombuffer(e, np.float32)[:2]).all() and np.isnan(np.frombuffer(v, np.float32)).all()
        assert (np.frombuffer(i, np.int32) == -1).all()
        with pytest.raises(RuntimeError, match="status 2"):
            rt.synchronize()
        again()
        assert answers() == want


def test_refusals(rt):
    put(rt, "l", np.zeros((2, 50), np.float32))
    put(rt, "h", np.zeros((2, 50), np.float16))
    put(rt, "t", np.zeros(2, np.int32))
    put(rt, "o", np.zeros(2, np.float32))
    put(rt, "e", np.zeros(2, np.float32))
    put(rt, "i", np.zeros(8, np.int32))
    put(rt, "v", np.zeros(8, np.float32))
    rt.alloc("b", 200, 1)
    ok = dict(logits="l", tokens="t", vocab=50, rows=2, out="o", entropy="e", top=4, top_ids="i", top_out="v")
    rt.logprobs(**ok)
    rt.logprobs(**{**ok, "logits": "h"})
    for bad, error in ((dict(vocab=0), ValueError), (dict(vocab=51), ValueError), (dict(vocab=(1 << 30) + 1), ValueError), (dict(rows=0), ValueError), (dict(rows=3), ValueError), (dict(top=-1), ValueError),
                       (dict(top=33), ValueError), (dict(top=5), ValueError), (dict(top_ids=None), ValueError), (dict(top=0), ValueError), (dict(top=0, top_ids=None), ValueError),
                       (dict(logits="b"), TypeError), (dict(out="h"), TypeError), (dict(logits="nothing"), KeyError), (dict(tokens="h"), TypeError), (dict(temperature="h"), TypeError),
                       (dict(out="t"), ValueError), (dict(entropy="o"), ValueError), (dict(top_out="i"), ValueError), (dict(out="l"), ValueError), (dict(entropy="l"), ValueError),
                       (dict(top_ids="l"), ValueError), (dict(temperature="o"), ValueError), (dict(top_out="l"), ValueError), (dict(temperature="e"), ValueError)):
        with pytest.raises(error):
            rt.logprobs(**{**ok, **bad})
    rt.logprobs("l", "t", 50, 2, out="o")  # no alternatives, no entropy
