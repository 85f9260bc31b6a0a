"""The passes in 8-bit floating point and the log probabilities together, as a scoring pass uses them: norm -> gate / up -> silu * up -> down onto the residual -> norm ->
LM head -> log probabilities of the tokens that follow; step by step against the formulas, eagerly, captured and replayed, on another stream, in two runtimes at once, beside
the other passes of the library."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

from tests import f8_formulas as F
from tests.test_gpu_f8 import GATE, NORM, bound
from vinf_3080ti_b200.gguf_types import GGUFTensorType as T
from vinf_3080ti_b200.synth import synthetic_blocks

pytestmark = pytest.mark.gpu

HIDDEN, FFN, VOCAB, TOP = 512, 1280, 2004, 5


class Pass:
    """A layer's FFN and the LM head, weights converted from GGUF blocks."""

    def __init__(self, codebooks, seed=0, ntok=12, kind=np.float32):
        from vinf_3080ti_b200.runtime import Runtime

        self.rt = rt = Runtime(codebooks["iq3s_grid"], codebooks)
        self.n = n = ntok
        rng = np.random.default_rng(seed)
        self.w = {}
        for name, t, rows, cols in (("gate", T.Q4_K, FFN, HIDDEN), ("up", T.Q4_K, FFN, HIDDEN), ("down", T.Q6_K, HIDDEN, FFN), ("head", T.Q8_0, VOCAB, HIDDEN)):
            rt.upload(name, synthetic_blocks(t, rows, cols, rng, 1e-4, 1e-3), int(t), cols, rows)
            rt.convert_f8(name, name)
            addr, _, _, _, pitch, _, _ = rt.tensor_info(name)
            at = (rows * pitch + 255) // 256 * 256
            rt.bind("raw", addr, at + 4 * F.blocks(rows) * F.blocks(cols), 1)
            raw = rt.read_array("raw").view(np.uint8)
            rt.release("raw")
            self.w[name] = raw[:rows * pitch].reshape(rows, pitch)[:, :cols].copy(), raw[at:].view(np.float32).reshape(F.blocks(rows), F.blocks(cols)).copy()
        elem = np.dtype(kind).itemsize
        for name, count, e in (("delta", n * HIDDEN, elem), ("h", n * HIDDEN, elem), ("gate_y", n * FFN, elem), ("up_y", n * FFN, elem), ("q", n * HIDDEN, 1),
                               ("s", F.blocks(HIDDEN) * F.scale_pitch(n), 4), ("q2", n * FFN, 1), ("s2", F.blocks(FFN) * F.scale_pitch(n), 4), ("g", HIDDEN, 4), ("logits", n * VOCAB, elem),
                               ("tokens", n, 4), ("lp", n, 4), ("entropy", n, 4), ("ids", n * TOP, 4), ("best", n * TOP, 4)):
            rt.alloc(name, count, e)
        self.data = {"delta": rng.standard_normal((n, HIDDEN)).astype(kind), "h": (rng.standard_normal((n, HIDDEN)) * 2).astype(kind),
                     "g": rng.uniform(0.5, 1.5, HIDDEN).astype(np.float32), "tokens": rng.integers(0, VOCAB, n).astype(np.int32)}
        self.kind = kind
        self.reset()

    def reset(self):
        for name, a in self.data.items():
            self.rt.write(name, a)

    def steps(self):
        rt, n = self.rt, self.n
        yield lambda: rt.rows_f8("delta", "q", "s", HIDDEN, n, residual="h", norm="g")
        yield lambda: rt.qmm_f8("gate", "q", "s", "gate_y", n)
        yield lambda: rt.qmm_f8("up", "q", "s", "up_y", n)
        yield lambda: rt.rows_f8("gate_y", "q2", "s2", FFN, n, silu_mul="up_y")
        yield lambda: rt.qmm_f8("down", "q2", "s2", "h", n, add=True)
        yield lambda: rt.rows_f8("h", "q", "s", HIDDEN, n, norm="g")
        yield lambda: rt.qmm_f8("head", "q", "s", "logits", n)
        yield lambda: rt.logprobs("logits", "tokens", VOCAB, n, out="lp", entropy="entropy", top=TOP, top_ids="ids", top_out="best")

    def run(self):
        for step in self.steps():
            step()

    def seen(self):
        return {name: self.rt.read(name) for name in ("h", "gate_y", "up_y", "q", "q2", "logits", "lp", "entropy", "ids", "best")}

    def rows(self, q, s, cols):
        return (self.rt.read_array(q).view(np.uint8).reshape(self.n, cols), self.rt.read_array(s).reshape(F.blocks(cols), -1)[:, :self.n])


def near_rows(got, n, off):
    """Scales and e4m3 values against n in 64 bits, as the tolerances of the single calls have it."""
    q, s = got
    want = F.scales_of(n)
    assert (np.abs(s - want) <= (off + F.U) * 1.01 * want).all()
    t = n / F.spread_scales(s.astype(np.float64), n.shape[1])
    assert (np.abs(F.CODES[q] - t) <= F.step(t * (1 + off)) / 2 + np.abs(t) * (off + 2 * F.U) * 1.01).all()


@pytest.mark.parametrize("ntok", [1, 12, 70, 150])
@pytest.mark.parametrize("kind", [np.float32, np.float16])
def test_every_step_of_a_pass(codebooks, kind, ntok):
    p = Pass(codebooks, ntok=ntok, kind=kind)
    rt, d = p.rt, p.data
    steps = list(p.steps())

    def product(name, q, s, got, before=0.0):
        want, most = F.qmm(*p.w[name], q, s)
        want, most = want + before, most + np.abs(before)
        assert (np.abs(got - want) <= bound(most, want, q.shape[1], kind)).all()

    steps[0]()
    n, h = F.values(d["delta"], residual=d["h"], norm=d["g"])
    assert np.array_equal(rt.read_array("h").reshape(ntok, HIDDEN), h)
    q, s = p.rows("q", "s", HIDDEN)
    near_rows((q, s), n, NORM)
    steps[1]()
    steps[2]()
    gate, up = (rt.read_array(name).reshape(ntok, FFN) for name in ("gate_y", "up_y"))
    product("gate", q, s, gate)
    product("up", q, s, up)
    steps[3]()
    q2, s2 = p.rows("q2", "s2", FFN)
    near_rows((q2, s2), F.values(gate, x2=up)[0], GATE)
    steps[4]()
    h2 = rt.read_array("h").reshape(ntok, HIDDEN)
    product("down", q2, s2, h2, h.astype(np.float64))
    steps[5]()
    q, s = p.rows("q", "s", HIDDEN)
    near_rows((q, s), F.values(h2, norm=d["g"])[0], NORM)
    steps[6]()
    logits = rt.read_array("logits").reshape(ntok, VOCAB)
    assert np.isfinite(logits).all()
    product("head", q, s, logits)
    steps[7]()
    lp, entropy, ids, best = F.logprobs(logits, d["tokens"], TOP)
    assert np.array_equal(np.frombuffer(rt.read("ids"), np.int32).reshape(ntok, TOP), ids)
    sums = (4 * entropy + 4 + 16 + 7 * (VOCAB / 8192 + 1) + 22) * F.U
    assert (np.abs(rt.read_array("lp") - lp) <= sums + 3 * F.U * np.abs(lp)).all() and (np.abs(rt.read_array("entropy") - entropy) <= sums * (1 + 3 * entropy)).all()
    assert (np.abs(rt.read_array("best").reshape(ntok, TOP) - best) <= sums[:, None] + 3 * F.U * np.abs(best)).all()
    # the same as one run without waits
    first = p.seen()
    p.reset()
    p.run()
    assert p.seen() == first
    rt.close()


@pytest.mark.parametrize("ntok", [1, 12, 150])
def test_captured_and_replayed(codebooks, ntok):
    p = Pass(codebooks, 1, ntok)
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
        assert p.seen() == want
    assert rt.launch_count() - before >= 3 * 8
    # replays back to back: h grows from pass to pass, exactly as eager passes make it grow
    p.reset()
    for _ in range(3):
        p.run()
    want = p.seen()
    p.reset()
    for g in (graphs[1], graphs[0], graphs[1]):
        rt.graph_launch(g)
    assert p.seen() == want
    for g in graphs:
        rt.graph_destroy(g)
    rt.close()


def test_on_another_stream(codebooks):
    import torch

    p = Pass(codebooks, 2, 20)
    p.run()
    want = p.seen()
    stream = torch.cuda.Stream()
    p.rt.set_stream(stream.cuda_stream)
    p.reset()
    p.run()
    assert p.seen() == want
    p.rt.set_stream(None)
    p.reset()
    p.run()
    assert p.seen() == want
    p.rt.close()


def test_runtimes_at_once(codebooks):
    """Their launches overlap on the GPU; of few rows, of many, of both."""
    passes = [Pass(codebooks, 3, 4), Pass(codebooks, 4, 300), Pass(codebooks, 5, 40)]
    for p in passes:
        for _ in range(20):
            p.run()
    together = [p.seen() for p in passes]
    for p, want in zip(passes, together):  # the same number of passes, one runtime after the other
        p.reset()
        for _ in range(20):
            p.run()
        assert p.seen() == want
        p.rt.close()


@pytest.mark.parametrize("ntok", [1, 24, 60, 200])
def test_between_the_other_passes_of_the_library(codebooks, ntok):
    """Launches of every kind in one stream, each reading what the one before has written; they begin before it has ended and share SMs and tensor memory with it."""
    from vinf_3080ti_b200.runtime import Runtime

    rt = Runtime(codebooks["iq3s_grid"], codebooks)
    rng = np.random.default_rng(6)
    rows, cols = 2048, 1024
    rt.upload("a", synthetic_blocks(T.Q4_K, rows, cols, rng, 1e-4, 1e-3), int(T.Q4_K), cols, rows)
    rt.upload("b", synthetic_blocks(T.Q4_K, cols, rows, rng, 1e-4, 1e-3), int(T.Q4_K), rows, cols)
    rt.convert_i8("b", "b8")
    rt.convert_f8("a", "af")
    rt.convert_f8("b", "bf")
    for name, n, e in (("x", ntok * cols, 4), ("y", ntok * rows, 4), ("q", ntok * rows, 1), ("s", ntok * 16 + 64, 4), ("z", ntok * cols, 4), ("y2", ntok * rows, 4), ("t", ntok, 4), ("lp", ntok, 4)):
        rt.alloc(name, n, e)
    rt.write("x", rng.standard_normal((ntok, cols)).astype(np.float32))

    def go(wait):
        for _ in range(1 if wait else 10):
            for call in (lambda: rt.rows_f8("x", "q", "s", cols, ntok), lambda: rt.qmm_f8("af", "q", "s", "y", ntok), lambda: rt.rows_i8("y", "q", "s", rows, ntok),
                         lambda: rt.qmm_i8("b8", "q", "s", "z", ntok), lambda: rt.qmv("a", "z", "y2", ntok), lambda: rt.rows_f8("y2", "q", "s", rows, ntok),
                         lambda: rt.qmm_f8("bf", "q", "s", "z", ntok), lambda: rt.logprobs("z", "t", cols, ntok, out="lp")):
                call()
                if wait:
                    rt.synchronize()
        return [rt.read(n) for n in ("y", "z", "y2", "lp")]

    want = go(True)
    assert go(False) == want
    rt.capture_begin()
    for _ in range(5):
        rt.rows_f8("x", "q", "s", cols, ntok)
        rt.qmm_f8("af", "q", "s", "y", ntok)
        rt.qmv("a", "x", "y2", min(ntok, 8))
        rt.qmm_f8("af", "q", "s", "y", ntok)
    graph = rt.capture_end()
    rt.zero("y")
    rt.graph_launch(graph)
    assert rt.read("y") == want[0]
    rt.graph_destroy(graph)
    rt.close()


RUN_IN_A_PROCESS = """
import hashlib
import sys
import numpy as np
sys.path.insert(0, {repo!r})
from vinf_3080ti_b200.runtime import Runtime
rt = Runtime()
rng = np.random.default_rng(0)
cols, vocab, most = 640, 40000, 300
w = rng.integers(0, 0x78, (vocab, cols), dtype=np.uint8)
rt.upload_f8("w", w, np.full((313, 5), 1e-4, np.float32), cols, vocab)
rt.upload_f8("few", w[:300], np.full((3, 5), 1e-4, np.float32), cols, 300)
for name, n, e in (("x", most * cols, 4), ("g", cols, 4), ("q", most * cols, 1), ("s", 5 * most, 4), ("y", most * 300, 4), ("logits", 4 * vocab, 4), ("k", 4, 4), ("out", 4, 4), ("ids", 80, 4)):
    rt.alloc(name, n, e)
rt.write("x", rng.standard_normal((most, cols)).astype(np.float32))
rt.write("g", np.ones(cols, np.float32))
def go():
    for ntok in (2, 20, 50, 100, most):
        rt.rows_f8("x", "q", "s", cols, ntok, norm="g")
        rt.qmm_f8("few", "q", "s", "y", ntok)
    rt.rows_f8("x", "q", "s", cols, 4)
    rt.qmm_f8("w", "q", "s", "logits", 4)
    rt.logprobs("logits", "k", vocab, 4, out="out", top=20, top_ids="ids")
names = ("q", "s", "y", "logits", "out", "ids")
if {capture}:
    rt.capture_begin()
    go()
    graph = rt.capture_end()
    rt.graph_launch(graph)
    first = [rt.read(n) for n in names]
    for n in names:
        rt.zero(n)
    go()
    assert first == [rt.read(n) for n in names]
else:
    go()
rt.synchronize()
print(hashlib.sha256(b"".join(rt.read(n) for n in names)).hexdigest())
"""


def run_in_a_process(capture, **env):
    import os

    repo = str(Path(__file__).resolve().parent.parent)
    done = subprocess.run([sys.executable, "-c", RUN_IN_A_PROCESS.format(repo=repo, capture=capture)], capture_output=True, text=True, timeout=300, env={**os.environ, **env})
    assert done.returncode == 0, done.stderr[-2000:]
    return done.stdout.strip()


def test_the_first_calls_of_a_process_may_be_captured_and_launches_need_not_overlap():
    want = run_in_a_process(True)
    assert len(want) == 64
    assert run_in_a_process(False) == want
    assert run_in_a_process(False, VINF_B200_NO_PDL="1") == want


def test_replacing_a_tensor_beside_a_capture():
    import torch

    from vinf_3080ti_b200.runtime import Runtime

    rt = Runtime()
    one = int(F.encode(1.0))
    w, s = torch.full((4, 48), one, dtype=torch.uint8, device="cuda"), torch.ones(1, device="cuda")
    torch.cuda.synchronize()
    rt.upload_f8("mine", np.full((4, 48), F.encode(2.0), np.uint8), np.ones((1, 1), np.float32), 48, 4)
    rt.bind_f8("bound", w.data_ptr(), s.data_ptr(), 48, 4)
    for name, n, elem in (("q", 48, 1), ("s", 4, 4), ("y", 4, 4), ("y2", 4, 4)):
        rt.alloc(name, n, elem)
    rt.write("q", np.full(48, one, np.uint8))
    rt.write("s", np.ones(4, np.float32))
    rt.capture_begin()
    rt.qmm_f8("mine", "q", "s", "y")
    for name in ("mine", "bound"):
        with pytest.raises(ValueError, match="captured"):
            rt.bind_f8(name, w.data_ptr(), s.data_ptr(), 48, 4)
    for call in (lambda: rt.upload_f8("x", np.zeros((4, 48), np.uint8), np.ones((1, 1), np.float32), 48, 4), lambda: rt.upload_f8("mine", np.zeros((4, 48), np.uint8), np.ones((1, 1), np.float32), 48, 4)):
        with pytest.raises(ValueError, match="captured"):
            call()
    rt.bind_f8("new", w.data_ptr(), s.data_ptr(), 48, 4)
    rt.qmm_f8("new", "q", "s", "y2")
    graph = rt.capture_end()
    rt.graph_launch(graph)
    assert rt.read_array("y").tolist() == [96.0] * 4 and rt.read_array("y2").tolist() == [48.0] * 4
    rt.bind_f8("bound", w.data_ptr(), s.data_ptr(), 48, 3)  # afterwards it may be replaced
    assert rt.tensor_info("bound")[2:4] == (3, 48)
    rt.graph_destroy(graph)
    rt.close()
