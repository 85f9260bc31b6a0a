"""The 8-bit passes and the verification together, as a verification pass of speculative decoding uses them: norm -> gate / up -> silu * up -> down onto
the residual -> norm -> LM head -> verify; eagerly, captured into a graph and replayed, on another stream, in two runtimes at once."""
from __future__ import annotations

import numpy as np
import pytest

from tests import i8_formulas as F
from vinf_3080ti_b200.gguf_types import GGUFTensorType as T
from vinf_3080ti_b200.synth import synthetic_blocks

pytestmark = pytest.mark.gpu

HIDDEN, FFN, VOCAB, SEQS, DRAFTS = 512, 1280, 1999, 3, 3
NTOK = SEQS * (DRAFTS + 1)


class Pass:
    """A layer's FFN and the LM head, weights converted from GGUF blocks."""

    def __init__(self, codebooks, seed=0, kind=np.float32, gain=1.0):
        from vinf_3080ti_b200.runtime import Runtime

        self.rt = rt = Runtime(codebooks["iq3s_grid"], codebooks)
        self.kind = kind
        rng = np.random.default_rng(seed)
        self.w = {}
        for name, t, rows, cols in (("gate", T.Q4_K, FFN, HIDDEN), ("up", T.Q4_K, FFN, HIDDEN), ("down", T.Q6_K, HIDDEN, FFN), ("head", T.Q8_0, VOCAB, HIDDEN)):
            rt.upload(name, synthetic_blocks(t, rows, cols, rng), int(t), cols, rows)
            rt.alloc("full", rows * cols)
            rt.dequantize(name, "full")
            self.w[name] = F.rows_i8(rt.read_array("full").reshape(rows, cols))[:2]
            rt.convert_i8(name, name)
        elem = np.dtype(kind).itemsize
        for name, n, e in (("delta", NTOK * HIDDEN, elem), ("h", NTOK * HIDDEN, elem), ("gate_y", NTOK * FFN, elem), ("up_y", NTOK * FFN, elem), ("q", NTOK * FFN, 1), ("s", NTOK, 4),
                           ("q2", NTOK * FFN, 1), ("s2", NTOK, 4), ("g", HIDDEN, 4), ("logits", NTOK * VOCAB, elem), ("tokens", SEQS * DRAFTS, 4), ("u", SEQS * (DRAFTS + 1), 4),
                           ("out", SEQS * (DRAFTS + 2), 4)):
            rt.alloc(name, n, e)
        self.data = {"delta": rng.standard_normal((NTOK, HIDDEN)).astype(kind), "h": (rng.standard_normal((NTOK, HIDDEN)) * 2).astype(kind),
                     "g": (gain * rng.uniform(0.5, 1.5, HIDDEN)).astype(np.float32), "u": rng.random((SEQS, DRAFTS + 1), dtype=np.float32),
                     "tokens": rng.integers(0, VOCAB, (SEQS, DRAFTS)).astype(np.int32)}
        self.reset()

    def reset(self):
        for name, a in self.data.items():
            self.rt.write(name, a)

    def run(self):
        rt = self.rt
        rt.rows_i8("delta", "q", "s", HIDDEN, NTOK, residual="h", norm="g")
        rt.qmm_i8("gate", "q", "s", "gate_y", NTOK)
        rt.qmm_i8("up", "q", "s", "up_y", NTOK)
        rt.rows_i8("gate_y", "q2", "s2", FFN, NTOK, silu_mul="up_y")
        rt.qmm_i8("down", "q2", "s2", "h", NTOK, add=True)
        rt.rows_i8("h", "q", "s", HIDDEN, NTOK, norm="g")
        rt.qmm_i8("head", "q", "s", "logits", NTOK)
        rt.verify("logits", None, "tokens", "u", VOCAB, SEQS, DRAFTS, out="out", blocking=False)

    def seen(self):
        return {n: self.rt.read_array(n).copy() for n in ("h", "gate_y", "up_y", "q", "q2", "s", "s2", "logits")} | {"out": np.frombuffer(self.rt.read("out"), np.int32).copy()}


@pytest.mark.parametrize("kind,gain", [(np.float32, 1.0), (np.float16, 1.0), (np.float16, 2.0**-7)], ids=["fp32", "fp16-that-overflows", "fp16"])
def test_every_step_of_a_pass(codebooks, kind, gain):
    p = Pass(codebooks, kind=kind, gain=gain)
    rt, d = p.rt, p.data
    last = 2.0**-11 * 1.01 if kind is np.float16 else 0.0

    def near(got, want, extra=0.0):
        with np.errstate(all="ignore"):
            limit = 3.03 * 2.0**-24 * np.abs(want) + last * np.abs(want) + 2.0**-25 + extra
            ends = np.isnan(want) & np.isnan(got) | (kind is np.float16) & (np.abs(want) >= 65520 - limit) & (np.abs(want) * np.sign(got) == want) & np.isinf(got)
            return (ends | (np.abs(got.astype(np.float64) - want) <= limit)).all()

    rt.rows_i8("delta", "q", "s", HIDDEN, NTOK, residual="h", norm="g")
    q, s, h = F.rows_i8(d["delta"], residual=d["h"], norm=d["g"])
    assert np.array_equal(rt.read_array("q")[:NTOK * HIDDEN].reshape(NTOK, HIDDEN), q) and np.array_equal(rt.read_array("s"), s)
    assert np.array_equal(rt.read_array("h").reshape(NTOK, HIDDEN), h)
    rt.qmm_i8("gate", "q", "s", "gate_y", NTOK)
    rt.qmm_i8("up", "q", "s", "up_y", NTOK)
    gate, up = (rt.read_array(n).reshape(NTOK, FFN) for n in ("gate_y", "up_y"))
    assert near(gate, F.qmm_i8(*p.w["gate"], q, s)[0]) and near(up, F.qmm_i8(*p.w["up"], q, s)[0])
    rt.rows_i8("gate_y", "q2", "s2", FFN, NTOK, silu_mul="up_y")
    q2, s2, _ = F.rows_i8(gate, x2=up)
    assert np.array_equal(rt.read_array("q2").reshape(NTOK, FFN), q2) and np.array_equal(rt.read_array("s2"), s2, equal_nan=True)
    assert gain == 1.0 or np.isfinite(s2).all()
    rt.qmm_i8("down", "q2", "s2", "h", NTOK, add=True)
    down = F.qmm_i8(*p.w["down"], q2, s2)[0]
    h2 = rt.read_array("h").reshape(NTOK, HIDDEN)
    assert near(h2, h + down, 4.04 * 2.0**-24 * np.abs(down))
    rt.rows_i8("h", "q", "s", HIDDEN, NTOK, norm="g")
    q, s, _ = F.rows_i8(h2, norm=d["g"])
    rt.qmm_i8("head", "q", "s", "logits", NTOK)
    logits = rt.read_array("logits").reshape(NTOK, VOCAB)
    assert (kind is np.float16 and gain == 1.0) or np.isfinite(logits).all()
    assert near(logits, F.qmm_i8(*p.w["head"], q, s)[0])
    # drafts that are likely to be kept
    p.data["tokens"] = logits.reshape(SEQS, DRAFTS + 1, VOCAB)[:, :DRAFTS].argmax(-1).astype(np.int32)
    rt.write("tokens", p.data["tokens"])
    kept = rt.verify("logits", None, "tokens", "u", VOCAB, SEQS, DRAFTS, out="out")
    want = F.verify(logits.reshape(SEQS, DRAFTS + 1, VOCAB), None, p.data["tokens"], d["u"])
    assert kept == [list(r[1:r[0] + 2]) for r in want]
    # the same as one run without waits
    first = p.seen()
    p.reset()
    p.run()
    again = p.seen()
    assert all(np.array_equal(first[n], again[n], equal_nan=n != "out") for n in first)
    rt.close()


def equal(a, b):
    return all(np.array_equal(a[n], b[n]) for n in a)


def test_captured_and_replayed(codebooks):
    p = Pass(codebooks, 1)
    rt = p.rt
    p.run()
    want = p.seen()
    graphs = []
    for _ in range(2):  # two graphs of the same pass
        rt.capture_begin()
        p.run()
        graphs.append(rt.capture_end())
    before = rt.launch_count()
    for g in (*graphs, graphs[0]):
        p.reset()
        rt.graph_launch(g)
        assert equal(p.seen(), want)
    assert rt.launch_count() - before >= 3 * 8
    # replays back to back: h grows from pass to pass, exactly as eager passes make it grow
    p.reset()
    for _ in range(3):
        p.run()
    want = p.seen()
    p.reset()
    for g in (graphs[1], graphs[0], graphs[1]):
        rt.graph_launch(g)
    assert equal(p.seen(), want)
    for g in graphs:
        rt.graph_destroy(g)
    rt.close()


def test_on_another_stream(codebooks):
    import torch

    p = Pass(codebooks, 2)
    p.run()
    want = p.seen()
    stream = torch.cuda.Stream()
    p.rt.set_stream(stream.cuda_stream)
    p.reset()
    p.run()
    assert equal(p.seen(), want)
    p.rt.set_stream(None)
    p.reset()
    p.run()
    assert equal(p.seen(), want)
    p.rt.close()


def test_two_runtimes_at_once(codebooks):
    a, b = Pass(codebooks, 3), Pass(codebooks, 4)
    wants = []
    for p in (a, b):
        p.run()
        wants.append(p.seen())
        p.reset()
    for _ in range(20):
        for p in (a, b):
            p.run()
    for p in (a, b):  # the same number of passes, one runtime after the other
        together = p.seen()
        p.reset()
        for _ in range(20):
            p.run()
        assert equal(p.seen(), together)
        p.reset()
        p.run()
    assert equal(a.seen(), wants[0]) and equal(b.seen(), wants[1])
    a.rt.close()
    b.rt.close()


def test_between_matvecs_of_gguf_blocks(codebooks):
    """Launches of both kinds in one stream, each reading what the one before has written."""
    from vinf_3080ti_b200.runtime import Runtime

    rt = Runtime(codebooks["iq3s_grid"], codebooks)
    rng = np.random.default_rng(5)
    rt.upload("a", synthetic_blocks(T.Q4_K, 2048, 1024, rng), int(T.Q4_K), 1024, 2048)
    rt.upload("b", synthetic_blocks(T.Q4_K, 1024, 2048, rng), int(T.Q4_K), 2048, 1024)
    rt.convert_i8("b", "b8")
    for name, n, e in (("x", 4 * 1024, 4), ("y", 4 * 2048, 4), ("q", 4 * 2048, 1), ("s", 4, 4), ("z", 4 * 1024, 4), ("y2", 4 * 2048, 4)):
        rt.alloc(name, n, e)
    rt.write("x", rng.standard_normal((4, 1024)).astype(np.float32))

    def go(wait):
        for call in (lambda: rt.qmv("a", "x", "y", 4), lambda: rt.rows_i8("y", "q", "s", 2048, 4), lambda: rt.qmm_i8("b8", "q", "s", "z", 4), lambda: rt.qmv("a", "z", "y2", 4)):
            call()
            if wait:
                rt.synchronize()
        return rt.read_array("y2").copy()

    want = go(True)
    for _ in range(30):
        rt.zero("y")
        rt.zero("z")
        assert np.array_equal(go(False), want)
    rt.close()


@pytest.mark.parametrize("ntok", [1, 8, 24])
def test_products_and_matvecs_that_begin_before_the_last_one_ends(codebooks, ntok):
    """Captured products of few rows and matvecs by turns: blocks of two launches share SMs and their tensor memory."""
    from vinf_3080ti_b200.runtime import Runtime

    rt = Runtime(codebooks["iq3s_grid"], codebooks)
    rng = np.random.default_rng(6)
    rt.upload("a", synthetic_blocks(T.Q4_K, 2048, 1024, rng), int(T.Q4_K), 1024, 2048)
    for name, rows in (("few", 384), ("many", 19000)):
        w = rng.integers(-127, 128, (rows, 1024), dtype=np.int8)
        rt.upload_i8(name, w, np.full(rows, 1e-3, np.float32), 1024, rows)
    for name, n, e in (("x", ntok * 1024, 4), ("q", ntok * 1024, 1), ("s", ntok, 4), ("y", ntok * 2048, 4), ("few_y", ntok * 384, 4), ("many_y", ntok * 19000, 4)):
        rt.alloc(name, n, e)
    rt.write("x", rng.standard_normal((ntok, 1024)).astype(np.float32))
    rt.rows_i8("x", "q", "s", 1024, ntok)

    def go(wait):
        for _ in range(1 if wait else 25):
            for call in (lambda: rt.qmm_i8("few", "q", "s", "few_y", ntok), lambda: rt.qmv("a", "x", "y", ntok), lambda: rt.qmm_i8("many", "q", "s", "many_y", ntok),
                         lambda: rt.qmv("a", "x", "y", ntok)):
                call()
                if wait:
                    rt.synchronize()

    def seen():
        return [rt.read(n) for n in ("y", "few_y", "many_y")]

    go(True)
    want = seen()
    rt.capture_begin()
    go(False)
    graph = rt.capture_end()
    for _ in range(4):
        for n in ("y", "few_y", "many_y"):
            rt.zero(n)
        rt.graph_launch(graph)
        assert seen() == want
    rt.graph_destroy(graph)
    rt.close()


FIRST_IN_A_CAPTURE = """
import sys
import numpy as np
sys.path.insert(0, {repo!r})
from vinf_3080ti_b200.runtime import Runtime
rt = Runtime()
rng = np.random.default_rng(0)
cols, vocab = 640, 40000
w = rng.integers(-127, 128, (vocab, cols), dtype=np.int8)
rt.upload_i8("w", w, np.full(vocab, 1e-3, np.float32), cols, vocab)
rt.upload_i8("few", w[:300], np.full(300, 1e-3, np.float32), cols, 300)
for name, n, e in (("x", 300 * cols, 4), ("q", 300 * cols, 1), ("s", 300, 4), ("y", 300 * 300, 4), ("logits", 4 * vocab, 4), ("u", 4, 4), ("k", 3, 4), ("out", 5, 4)):
    rt.alloc(name, n, e)
rt.write("x", rng.standard_normal((300, cols)).astype(np.float32))
def go():
    for ntok in (2, 300):
        rt.rows_i8("x", "q", "s", cols, ntok)
        rt.qmm_i8("few", "q", "s", "y", ntok)
    rt.qmm_i8("w", "q", "s", "logits", 4)
    rt.verify("logits", None, "k", "u", vocab, 1, 3, out="out", blocking=False)
rt.capture_begin()
go()
graph = rt.capture_end()
rt.graph_launch(graph)
first = [rt.read(n) for n in ("q", "s", "y", "logits", "out")]
for n in ("q", "s", "y", "logits", "out"):
    rt.zero(n)
go()
assert first == [rt.read(n) for n in ("q", "s", "y", "logits", "out")]
rt.synchronize()
"""


def test_the_first_calls_of_a_process_may_be_captured():
    import subprocess
    import sys
    from pathlib import Path

    repo = str(Path(__file__).resolve().parent.parent)
    done = subprocess.run([sys.executable, "-c", FIRST_IN_A_CAPTURE.format(repo=repo)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
