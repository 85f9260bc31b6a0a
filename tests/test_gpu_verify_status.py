"""A verification whose logits may be what an expired wait has left: the failure is reported by the call that would answer from them."""
from __future__ import annotations

import numpy as np
import pytest

from vinf_3080ti_b200.gguf_types import GGUFTensorType as T
from vinf_3080ti_b200.sharding import ExchangeLayout
from vinf_3080ti_b200.synth import synthetic_blocks

pytestmark = pytest.mark.gpu


@pytest.fixture()
def late(codebooks):
    """A runtime whose last matvec waits for a push that no rank makes (a bounded wait, which runs out)."""
    from vinf_3080ti_b200.runtime import Runtime

    layout = ExchangeLayout(4 * 64, n_slots=2)
    rts = [Runtime(codebooks["iq3s_grid"], codebooks) for _ in range(2)]
    addrs = [rt.exchange_create(layout.total)[1] for rt in rts]
    rt = rts[0]
    rt.exchange_config(0, addrs, layout.flag_off, layout.count_off, layout.n_slots)
    rt.upload("w", synthetic_blocks(T.Q8_0, 64, 256, np.random.default_rng(13)), int(T.Q8_0), 256, 64)
    rt.alloc("x", 256)
    rt.alloc("target", 2 * 64)
    for name, n in (("tokens", 1), ("u", 2), ("out", 3), ("out2", 3)):
        rt.alloc(name, n)
    rt.write("u", np.full(2, 0.5, np.float32))
    rt.qmv_push("w", "x", "target", 1, slot=1, dst_off=0, rows_total=64, row_begin=0)  # this rank pushes slot 1, the other never does
    rt.synchronize()

    def run_out():
        rt.qmv_push("w", "x", "target", 1, slot=-1, dst_off=0, rows_total=64, row_begin=0, wait_slot=1)

    yield rt, run_out
    for r in rts:
        r.close()


def verify(rt, **kw):
    return rt.verify("target", None, "tokens", "u", 64, 1, 1, **{"out": "out", **kw})


def test_a_blocking_call_reports_it_once(late):
    rt, run_out = late
    want = verify(rt)
    run_out()
    with pytest.raises(RuntimeError, match="status 2"):
        verify(rt)
    assert verify(rt) == want  # the runtime is usable again
    rt.synchronize()


def test_answers_that_are_not_waited_for_hold_no_tokens(late):
    rt, run_out = late
    want = verify(rt)
    run_out()
    verify(rt, blocking=False)
    verify(rt, out="out2", blocking=False)
    for name in ("out", "out2"):
        assert np.frombuffer(rt.read(name), np.int32).tolist() == [-1, -1, -1]
    with pytest.raises(RuntimeError, match="status 2"):
        rt.synchronize()
    assert verify(rt) == want


def test_replayed_answers_hold_no_tokens(late):
    rt, run_out = late
    want = verify(rt)
    rt.capture_begin()
    verify(rt, blocking=False)
    graph = rt.capture_end()
    run_out()
    rt.graph_launch(graph)
    assert np.frombuffer(rt.read("out"), np.int32).tolist() == [-1, -1, -1]
    with pytest.raises(RuntimeError, match="status 2"):
        rt.synchronize()
    rt.graph_launch(graph)
    got = np.frombuffer(rt.read("out"), np.int32)
    assert got[1:got[0] + 2].tolist() == want[0]
