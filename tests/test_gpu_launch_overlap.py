"""VINF_B200_NO_PDL=1 turns the overlap of launches off, for every kernel: weights that a kernel fills on the runtime's stream are then in place when
the next launch copies them.  Seen in the dependencies of a captured pass, and in the results of one whose weights are made just before."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from tests import i8_formulas as F
from vinf_3080ti_b200.gguf_types import GGUFTensorType as T

pytestmark = pytest.mark.gpu

FULL, PROGRAMMATIC = 0, 1


class EdgeData(ctypes.Structure):
    _fields_ = [("from_port", ctypes.c_uint8), ("to_port", ctypes.c_uint8), ("type", ctypes.c_uint8), ("reserved", ctypes.c_uint8 * 5)]


def edges_of(rt, calls):
    """Kinds of the dependencies between the launches of `calls`, captured on the runtime's stream (and not run)."""
    cu = ctypes.CDLL("libcuda.so.1")

    def check(status):
        assert status == 0, status

    stream, graph = ctypes.c_void_p(rt.stream()), ctypes.c_void_p()
    check(cu.cuStreamBeginCapture_v2(stream, 1))
    try:
        calls()
    finally:
        status = cu.cuStreamEndCapture(stream, ctypes.byref(graph))
    check(status)
    n = ctypes.c_size_t(0)
    check(cu.cuGraphGetEdges_v2(graph, None, None, None, ctypes.byref(n)))
    nodes, data = (ctypes.c_void_p * (2 * n.value))(), (EdgeData * n.value)()
    check(cu.cuGraphGetEdges_v2(graph, nodes, ctypes.byref(nodes, n.value * ctypes.sizeof(ctypes.c_void_p)), data, ctypes.byref(n)))
    kinds = [d.type for d in data[:n.value]]
    check(cu.cuGraphDestroy(graph))
    return kinds


@pytest.fixture(params=[False, True], ids=["overlap", "no-overlap"])
def made(request, codebooks, monkeypatch):
    from vinf_3080ti_b200.runtime import Runtime

    if request.param:
        monkeypatch.setenv("VINF_B200_NO_PDL", "1")
    else:
        monkeypatch.delenv("VINF_B200_NO_PDL", raising=False)
    rt = Runtime(codebooks["iq3s_grid"], codebooks)
    yield rt, request.param
    rt.synchronize()
    rt.close()


@pytest.mark.parametrize("rows,cols,ntok", [(300, 256, 3), (20000, 256, 20), (20000, 300, 300), (300, 2048, 300)], ids=["split", "tiles", "pairs", "pairs-split"])
def test_8_bit_passes(made, rows, cols, ntok):
    rt, off = made
    rt.upload_i8("w", np.ones((rows, cols), np.int8), np.ones(rows, np.float32), cols, rows)
    for name, n, elem in (("x", ntok * cols, 4), ("q", ntok * F.pitch(cols), 1), ("s", ntok, 4), ("y", ntok * rows, 4)):
        rt.alloc(name, n, elem)

    def calls():
        for _ in range(2):
            rt.rows_i8("x", "q", "s", cols, ntok)
            rt.qmm_i8("w", "q", "s", "y", ntok)

    assert edges_of(rt, calls) == [FULL if off else PROGRAMMATIC] * 3


@pytest.mark.parametrize("cols", [64, 67, 24576])
@pytest.mark.parametrize("gated", [False, True])
def test_every_form_of_rows(made, cols, gated):
    rt, off = made
    for name, n, elem in (("x", 2 * cols, 4), ("q", 2 * F.pitch(cols), 1), ("s", 2, 4), ("g", cols, 4)):
        rt.alloc(name, n, elem)

    def calls():
        for norm in (None, "g", None):
            rt.rows_i8("x", "q", "s", cols, 2, norm=norm, silu_mul="x" if gated else None)

    assert edges_of(rt, calls) == [FULL if off else PROGRAMMATIC] * 2


def test_verification(made):
    rt, off = made
    for name, n in (("target", 60), ("tokens", 4), ("u", 6), ("out", 8)):
        rt.alloc(name, n)

    def calls():
        for _ in range(3):
            rt.verify("target", None, "tokens", "u", 10, 2, 2, out="out", blocking=False)

    assert edges_of(rt, calls) == [FULL if off else PROGRAMMATIC] * 2


@pytest.mark.parametrize("t,cols,ntok", [(T.Q8_0, 256, 1), (T.Q4_K, 5120, 4), (T.F16, 256, 2), (T.Q4_K, 512, 70)], ids=["Q8_0", "Q4_K", "F16", "prompt"])
def test_matvecs_and_prompts(made, t, cols, ntok):
    from vinf_3080ti_b200.synth import synthetic_blocks

    rt, off = made
    rt.set_gemm_min_rows(64)
    rt.upload("w", synthetic_blocks(t, 512, cols, np.random.default_rng(1)), int(t), cols, 512)
    rt.alloc("x", ntok * cols)
    rt.alloc("y", ntok * 512)
    rt.qmv("w", "x", "y", ntok)  # (scratch of prompts is not allocated beside a capture)
    rt.synchronize()

    def calls():
        rt.qmv("w", "x", "y", ntok)
        rt.qmv("w", "x", "y", ntok)

    kinds = edges_of(rt, calls)
    assert len(kinds) == (3 if ntok == 70 else 1) and set(kinds) == {FULL if off else PROGRAMMATIC}


def test_weights_made_just_before_they_are_used(codebooks, monkeypatch):
    """A few rows of the weights take the slow way through 64 bits, so that they are written long after the launch has let its successor begin."""
    import torch

    from vinf_3080ti_b200.runtime import Runtime

    monkeypatch.setenv("VINF_B200_NO_PDL", "1")
    rt = Runtime(codebooks["iq3s_grid"], codebooks)
    rows, cols, ntok = 256, 20480, 2
    rng = np.random.default_rng(1)
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    x[[5, 77, 130, 255]] *= np.float32(1e-33)
    a = rng.standard_normal((ntok, cols)).astype(np.float32)
    w, ws, _ = F.rows_i8(x)
    q, qs, _ = F.rows_i8(a)
    want, _ = F.qmm_i8(w, ws, q, qs)
    xt, at = torch.from_numpy(x).cuda(), torch.from_numpy(a).cuda()
    wt, st = torch.empty((rows, cols), dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    torch.cuda.synchronize()
    rt.bind("x", xt.data_ptr(), xt.numel(), 4)
    rt.bind("a", at.data_ptr(), at.numel(), 4)
    rt.bind("wq", wt.data_ptr(), wt.numel(), 1)
    rt.bind("ws", st.data_ptr(), st.numel(), 4)
    rt.bind_i8("w", wt.data_ptr(), st.data_ptr(), cols, rows)
    rt.alloc("q", ntok * cols, 1)
    rt.alloc("s", ntok)
    rt.alloc("y", ntok * rows)
    rt.rows_i8("a", "q", "s", cols, ntok)
    for _ in range(5):
        wt.fill_(99)
        st.fill_(3.0)
        torch.cuda.synchronize()
        rt.rows_i8("x", "wq", "ws", cols, rows)
        rt.qmm_i8("w", "q", "s", "y", ntok)
        y = rt.read_array("y").reshape(ntok, rows)
        # three roundings of half a step (and those of subnormal products)
        off = np.abs(y - want) - 3 * 2.0**-24 * 1.01 * np.abs(want) - 2.0**-148
        assert (off <= 0).all(), np.unique(np.argwhere(off > 0)[:, 1])
    rt.close()
