"""Verification of drafted tokens on the GPU against its definition in 64 bits (tests/i8_formulas.py).  Tokens are whole numbers: they are equal."""
from __future__ import annotations

import numpy as np
import pytest

from tests import i8_formulas as F

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


def run(rt, target, draft, tokens, uniforms, lens=None, temperature=None):
    n, rows, vocab = target.shape
    k = rows - 1
    put(rt, "target", target)
    if draft is not None and k:
        put(rt, "draft", draft)
    if k:
        put(rt, "tokens", tokens.astype(np.int32))
    put(rt, "u", uniforms.astype(np.float32))
    if lens is not None:
        put(rt, "lens", lens.astype(np.int32))
    if temperature is not None:
        put(rt, "temp", temperature.astype(np.float32))
    put(rt, "out", np.full(n * (k + 2) + 3, 555, np.int32))
    kw = dict(out="out", lens=None if lens is None else "lens", temperature=None if temperature is None else "temp")
    args = ("target", "draft" if draft is not None and k else None, "tokens" if k else None, "u", vocab, n, k)
    kept = rt.verify(*args, **kw)
    raw = np.frombuffer(rt.read("out"), np.int32)
    assert (raw[n * (k + 2):] == 555).all()
    out = raw[:n * (k + 2)].reshape(n, k + 2)
    assert kept == [list(r[1:r[0] + 2]) for r in out]
    return out


def check(rt, target, draft, tokens, uniforms, **kw):
    got = run(rt, target, draft, tokens, uniforms, **kw)
    want = F.verify(target, draft, tokens, uniforms.astype(np.float32), **{n: v if n == "lens" else v.astype(np.float32) for n, v in kw.items()})
    assert np.array_equal(got, want), [(i, g.tolist(), w.tolist()) for i, (g, w) in enumerate(zip(got, want)) if (g != w).any()][:4]
    return got


def make(rng, n, k, vocab, kind=np.float32, spread=3.0, apart=0.7):
    target = (rng.standard_normal((n, k + 1, vocab)) * spread).astype(kind)
    draft = (target[:, :k] + apart * rng.standard_normal((n, k, vocab))).astype(kind)
    tokens = np.argmax(draft.astype(np.float32) + rng.gumbel(size=draft.shape), -1) if k else np.zeros((n, 0), int)
    return target, draft, tokens, rng.random((n, k + 1), dtype=np.float32)


VOCABS = [1, 2, 3, 5, 31, 32, 33, 127, 255, 1000, 1024, 4097, 8191, 32003, 151936]


@pytest.mark.parametrize("kind", [np.float32, np.float16])
@pytest.mark.parametrize("vocab", VOCABS)
def test_every_vocabulary(rt, vocab, kind):
    rng = np.random.default_rng(vocab)
    for n, k in ((1, 0), (1, 3), (3, 1), (5, 2)):
        target, draft, tokens, u = make(rng, n, k, vocab, kind)
        check(rt, target, draft, tokens, u)
        check(rt, target, None, tokens, u)


@pytest.mark.parametrize("n,k", [(1, 1), (2, 7), (7, 3), (13, 5), (40, 2), (75, 4), (150, 1), (310, 3), (2, 31), (1, 255)])
def test_batches(rt, n, k):
    rng = np.random.default_rng(n * 100 + k)
    target, draft, tokens, u = make(rng, n, k, 777, apart=0.4)
    lens = rng.integers(0, k + 1, n)
    temperature = rng.uniform(0.3, 1.5, n)
    got = check(rt, target, draft, tokens, u, lens=lens, temperature=temperature)
    assert (got[:, 0] <= lens).all()
    check(rt, target, None, tokens, u, lens=lens)
    check(rt, target, draft, tokens, u)


def test_large_batch_of_a_large_vocabulary(rt):
    rng = np.random.default_rng(0)
    target, draft, tokens, u = make(rng, 20, 3, 50257)
    got = check(rt, target, draft, tokens, u, temperature=rng.uniform(0.5, 1.2, 20))
    assert len(set(got[:, 0].tolist())) > 1


def test_drafts_equal_to_the_target_are_always_accepted(rt):
    rng = np.random.default_rng(1)
    target, _, tokens, u = make(rng, 9, 4, 3001)
    u[:, :-1] = np.float32(1 - 2.0**-24)
    got = check(rt, target, target[:, :4].copy(), tokens, u)
    assert (got[:, 0] == 4).all()


def test_random_numbers_at_their_ends(rt):
    rng = np.random.default_rng(2)
    target, draft, tokens, u = make(rng, 8, 2, 500)
    for value in (0.0, 2.0**-24, 1 - 2.0**-24):
        u[:] = np.float32(value)
        check(rt, target, draft, tokens, u)
        check(rt, target, None, tokens, u)


def test_greedy_verification_and_ties(rt):
    rng = np.random.default_rng(3)
    target = rng.integers(0, 4, (6, 4, 300)).astype(np.float32)  # many equal largest logits
    draft = target[:, :3].copy()
    draft[2:, 1] = rng.integers(0, 4, (4, 300))
    tokens = np.argmax(draft, -1)
    tokens[5, 0] = np.nonzero(target[5, 0] == 3)[0][1]  # as large, but not the first
    u = rng.random((6, 4), dtype=np.float32)
    for at in (0.0, -1.0, np.nan):
        got = check(rt, target, draft, tokens, u, temperature=np.full(6, at))
        assert got[0].tolist()[:4] == [3, *tokens[0]] and got[5, 0] == 0 and got[5, 1] == np.argmax(target[5, 0])
        check(rt, target, None, tokens, u, temperature=np.array([at, 1, at, 1, at, 1]))


def test_extreme_temperatures(rt):
    rng = np.random.default_rng(4)
    target, draft, tokens, u = make(rng, 6, 2, 640)
    for at in (1e-45, 1e-30, 1e-3, 100.0, 3e38, np.inf):
        check(rt, target, draft, tokens, u, temperature=np.full(6, at))


@pytest.mark.parametrize("kind", [np.float32, np.float16])
def test_masked_logits(rt, kind):
    rng = np.random.default_rng(5)
    target, draft, tokens, u = make(rng, 10, 3, 1500, kind)
    low = np.finfo(kind).min
    target[0, :, 100:] = -np.inf
    draft[0, :, 100:] = -np.inf
    target[1, :, ::2] = low
    draft[1, :, 1::2] = low
    target[2, 0, :] = -np.inf       # a mask that leaves nothing
    draft[3, 1, :] = -np.inf
    target[4, :, :] = -np.inf
    target[5, 1, 1499] = np.inf     # one certain token, two certain tokens
    target[6, 0, 3] = target[6, 0, 1400] = np.inf
    draft[6, 0, 3] = np.inf
    target[7, :, ::3] = np.nan
    draft[7, :, 1::3] = np.nan
    target[8, :, :] = low           # every logit the lowest value
    target[9, 3, :] = np.nan
    tokens = np.argmax(np.nan_to_num(draft.astype(np.float32), nan=-np.inf) + rng.gumbel(size=draft.shape), -1)
    tokens[6, 0] = 3
    for temperature in (None, np.full(10, 0.7), np.zeros(10)):
        kw = {} if temperature is None else {"temperature": temperature}
        got = check(rt, target, draft, tokens, u, **kw)
        assert got[4].tolist() == [0, -1, -1, -1, -1]
        check(rt, target, None, tokens, u, **kw)


def test_tokens_outside_the_vocabulary_are_refused(rt):
    rng = np.random.default_rng(6)
    target, draft, tokens, u = make(rng, 6, 3, 97, apart=0.0)
    tokens[0, 0], tokens[1, 1], tokens[2, 2], tokens[3, 0], tokens[4, 1] = -1, 97, 2**31 - 1, -2**31, 10**6
    got = check(rt, target, draft, tokens, u)
    assert got[:5, 0].tolist() == [0, 1, 2, 0, 1]
    check(rt, target, None, tokens, u)


def test_lengths_outside_their_range_are_clamped(rt):
    rng = np.random.default_rng(7)
    target, draft, tokens, u = make(rng, 5, 3, 64, apart=0.0)
    got = check(rt, target, draft, tokens, u, lens=np.array([-5, 0, 3, 4, 2**31 - 1]))
    assert got[:, 0].tolist() == [0, 0, 3, 3, 3]


def test_random_numbers_outside_their_range_do_no_harm(rt):
    rng = np.random.default_rng(8)
    target, draft, tokens, u = make(rng, 8, 2, 300)
    u[0], u[1], u[2], u[3], u[4] = 1.0, 5.0, -1.0, np.nan, np.inf
    got = run(rt, target, draft, tokens, u)
    assert ((got[:, 0] >= 0) & (got[:, 0] <= 2)).all()
    assert all(0 <= r[r[0] + 1] < 300 for r in got)


def test_tests_next_to_their_border(rt):
    """u q = p within fp32's last bits: 64 bits decide."""
    rng = np.random.default_rng(9)
    target, draft, tokens, _ = make(rng, 256, 1, 203, apart=1.5)
    ratio = np.array([F.spread(target[i, 0], 1.0)[tokens[i, 0]] / F.spread(draft[i, 0], 1.0)[tokens[i, 0]] for i in range(256)])
    some = np.nonzero(ratio < 0.99)[0]
    for step in (0, 1, -1):
        u = rng.random((256, 2), dtype=np.float32)
        near = ratio[some].astype(np.float32)
        u[some, 0] = near if step == 0 else np.nextafter(near, np.float32(step * 9))
        check(rt, target, draft, tokens, u)


def test_tokens_are_distributed_as_the_target(rt):
    """Rejection and the draw from the rest together give p: counts of 40000 sequences within five standard deviations."""
    rng = np.random.default_rng(10)
    n, vocab = 40000, 6
    target1, draft1 = rng.standard_normal((2, vocab)).astype(np.float32) * 1.5
    p, q = F.spread(target1, 1.0), F.spread(draft1, 1.0)
    tokens = rng.choice(vocab, size=(n, 1), p=q)
    out = run(rt, np.broadcast_to(target1, (n, 2, vocab)), np.broadcast_to(draft1, (n, 1, vocab)), tokens, rng.random((n, 2), dtype=np.float32))
    counts = np.bincount(out[:, 1], minlength=vocab)
    assert (np.abs(counts - n * p) <= 5 * np.sqrt(n * p * (1 - p))).all()


def test_rows_beyond_2_gi_elements(rt):
    """Offsets that pass 32 bits: 2.4e9 logits in 16 bits."""
    import torch

    n, k, vocab = 3900, 3, 152064
    target = torch.zeros((n, k + 1, vocab), dtype=torch.float16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(3)
    tokens = torch.randint(0, vocab, (n, k), generator=gen, device="cuda", dtype=torch.int32)
    target.scatter_(2, torch.cat([tokens, tokens[:, :1]], 1).long()[:, :, None], 30.0)  # each row is all but certain of its draft
    u = torch.full((n, k + 1), 0.5, device="cuda")
    out = torch.zeros((n, k + 2), dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    for name, t in (("big", target), ("bt", tokens), ("bu", u), ("bo", out)):
        rt.bind(name, t.data_ptr(), t.numel(), t.element_size())
    rt.verify("big", None, "bt", "bu", vocab, n, k, out="bo", blocking=False)
    rt.synchronize()
    assert torch.equal(out, torch.cat([torch.full_like(tokens[:, :1], k), tokens, tokens[:, :1]], 1))
    for name in ("big", "bt", "bu", "bo"):
        rt.release(name)


def test_refusals(rt):
    for name, n, elem in (("target", 2 * 3 * 10, 4), ("half", 60, 2), ("bytes", 60, 1), ("draft", 40, 4), ("tokens", 4, 4), ("u", 6, 4), ("out", 8, 4), ("two", 2, 4), ("one", 1, 4)):
        rt.alloc(name, n, elem)
    ok = dict(target="target", draft="draft", tokens="tokens", uniforms="u", vocab=10, seqs=2, drafts=2, out="out")
    rt.verify(**ok)
    for error, kw in ((ValueError, {"vocab": 0}), (ValueError, {"vocab": 11}), (ValueError, {"vocab": -1}), (ValueError, {"seqs": 0}), (ValueError, {"seqs": 3}), (ValueError, {"drafts": -1}),
                      (ValueError, {"drafts": 256}), (ValueError, {"drafts": 3}), (ValueError, {"tokens": None}), (ValueError, {"tokens": "two"}), (TypeError, {"tokens": "half"}),
                      (ValueError, {"uniforms": "two"}), (TypeError, {"uniforms": "half"}), (ValueError, {"out": "two"}), (TypeError, {"out": "half"}), (KeyError, {"target": "none"}),
                      (KeyError, {"draft": "none"}), (TypeError, {"draft": "half"}), (TypeError, {"target": "half"}), (TypeError, {"target": "bytes"}), (ValueError, {"draft": "two"}),
                      (ValueError, {"lens": "one"}), (TypeError, {"lens": "half"}), (ValueError, {"temperature": "one"}), (TypeError, {"temperature": "half"}), (KeyError, {"lens": "none"})):
        with pytest.raises(error):
            rt.verify(**{**ok, **kw})
    rt.verify(**{**ok, "lens": "two", "temperature": "two"})
    rt.capture_begin()
    try:
        with pytest.raises(ValueError):
            rt.verify(**ok)
        rt.verify(**ok, blocking=False)
    finally:
        rt.graph_destroy(rt.capture_end())


@pytest.mark.parametrize("name", ["target", "draft", "tokens", "u", "lens", "temp"])
def test_answers_have_a_buffer_of_their_own(rt, name):
    for buffer in ("target", "draft", "tokens", "u", "lens", "temp", "out"):
        rt.alloc(buffer, 60)
    with pytest.raises(ValueError, match="of their own"):
        rt.verify("target", "draft", "tokens", "u", 10, 2, 2, lens="lens", temperature="temp", out=name)
    rt.verify("target", "draft", "tokens", "u", 10, 2, 2, lens="lens", temperature="temp", out="out")
