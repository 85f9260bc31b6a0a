"""Memory that is written while other blocks still read it: refused whatever the names and types it goes by.  What only touches is not."""
from __future__ import annotations

import numpy as np
import pytest

from tests import i8_formulas as F

pytestmark = pytest.mark.gpu

COLS, NTOK, ROWS = 48, 3, 20


@pytest.fixture()
def memory():
    """A runtime and a function that binds names at offsets of one piece of memory."""
    import torch

    from vinf_3080ti_b200.runtime import Runtime

    rt = Runtime()
    room = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()

    def at(name, offset, n, elem=4):
        rt.bind(name, room.data_ptr() + offset, n, elem)

    n = NTOK * COLS
    for i, (name, count, elem) in enumerate((("x", n, 4), ("r", n, 4), ("t", n, 4), ("q", n, 1), ("s", NTOK, 4), ("g", COLS, 4), ("y", NTOK * ROWS, 4), ("h", n, 2), ("hr", n, 2))):
        at(name, 4096 * (i + 1), count, elem)
    rt.bind_i8("w", room.data_ptr() + 4096 * 12, room.data_ptr() + 4096 * 13, COLS, ROWS, pitch=64)
    at("weights", 4096 * 12, 1024)
    yield rt, at, room
    rt.synchronize()
    rt.close()


def rows(rt, **kw):
    a = dict(x="x", q="q", scales="s", cols=COLS, ntok=NTOK)
    a.update(kw)
    rt.rows_i8(a.pop("x"), a.pop("q"), a.pop("scales"), a.pop("cols"), a.pop("ntok"), **a)


@pytest.mark.parametrize("kw", [{}, {"norm": "g"}, {"residual": "r"}, {"residual": "r", "total": "x"}, {"residual": "r", "total": "t"}, {"residual": "x"}, {"silu_mul": "r"}, {"silu_mul": "x"},
                                {"x": "h"}, {"x": "h", "residual": "hr", "total": "h"}], ids=str)
def test_rows(memory, kw):
    rt, at, _ = memory
    rows(rt, **kw)  # apart
    elem = 2 if kw.get("x") == "h" else 4
    read = {kw.get("x", "x"), kw.get("residual"), kw.get("total"), kw.get("silu_mul"), kw.get("norm")} - {None}
    names = {"x": 1, "r": 2, "t": 3, "g": 6, "h": 8, "hr": 9}
    for name in read:
        size = COLS * 4 if name == "g" else NTOK * COLS * elem
        begin = 4096 * names[name]
        for offset, refused in ((0, True), (16, True), (size - 16, True), (size, False), (-NTOK * COLS, False), (16 - NTOK * COLS, True)):
            at("q2", begin + offset, NTOK * COLS, 1)
            if refused:
                with pytest.raises(ValueError, match="of their own"):
                    rows(rt, **{**kw, "q": "q2"})
            else:
                rows(rt, **{**kw, "q": "q2"})
        for offset, refused in ((0, True), (size - 16, True), (size, False), (-16, False)):
            at("s2", begin + offset, NTOK)
            if refused:
                with pytest.raises(ValueError, match="of their own"):
                    rows(rt, **{**kw, "scales": "s2"})
            else:
                rows(rt, **{**kw, "scales": "s2"})
    at("s2", 4096 * 4 + 16, NTOK)
    with pytest.raises(ValueError, match="of their own"):  # the scales among the 8-bit rows
        rows(rt, **{**kw, "scales": "s2"})


def test_sums_beside_what_they_are_made_of(memory):
    rt, at, _ = memory
    size = NTOK * COLS * 4
    for name, begin in (("x", 4096), ("r", 8192)):
        for offset, refused in ((0, False), (16, True), (-16, True), (size - 16, True), (size, False), (-size, False)):
            at("t2", begin + offset, NTOK * COLS)
            if refused:
                with pytest.raises(ValueError, match="of their own"):
                    rows(rt, residual="r", total="t2")
            else:
                rows(rt, residual="r", total="t2")
    at("x2", 4096, NTOK * COLS)  # another name of x
    rows(rt, residual="x", total="x2")
    rows(rt, x="x2", residual="x", total="x")
    at("t2", 4096 * 6 + COLS * 4 - 16, NTOK * COLS)
    with pytest.raises(ValueError, match="of their own"):
        rows(rt, residual="r", total="t2", norm="g")


def test_products(memory):
    rt, at, room = memory
    rng = np.random.default_rng(1)
    w, q = rng.integers(-128, 128, (ROWS, COLS), dtype=np.int8), rng.integers(-128, 128, (NTOK, COLS), dtype=np.int8)
    size = NTOK * ROWS * 4
    for begin, length in ((4096 * 4, NTOK * COLS), (4096 * 5, NTOK * 4), (4096 * 12, 64 * (ROWS - 1) + COLS), (4096 * 13, ROWS * 4)):
        end = (length + 15) // 16 * 16
        for offset, refused in ((0, True), (end - 16, True), (end, False), (-size, False), (16 - size, True)):
            at("y2", begin + offset, NTOK * ROWS)
            if refused:
                with pytest.raises(ValueError, match="of their own"):
                    rt.qmm_i8("w", "q", "s", "y2", NTOK)
            else:
                rt.qmm_i8("w", "q", "s", "y2", NTOK)
    # and what is apart still gives the product
    rt.synchronize()
    full = np.zeros((ROWS, 64), np.int8)
    full[:, :COLS] = w
    rt.write("weights", full.view(np.float32))
    at("ws", 4096 * 13, ROWS)
    rt.write("ws", np.ones(ROWS, np.float32))
    rt.write("q", q)
    rt.write("s", np.ones(NTOK, np.float32))
    rt.qmm_i8("w", "q", "s", "y", NTOK)
    assert np.array_equal(rt.read_array("y").reshape(NTOK, ROWS), F.qmm_i8(w, np.ones(ROWS), q, np.ones(NTOK))[0])


def test_answers_of_a_verification(memory):
    rt, at, _ = memory
    vocab, n, k = 10, 2, 2
    sizes = {"target": n * (k + 1) * vocab * 4, "draft": n * k * vocab * 4, "tokens": n * k * 4, "u": n * (k + 1) * 4, "lens": n * 4, "temp": n * 4}
    for i, (name, size) in enumerate(sizes.items()):
        at(name, 4096 * (i + 1), size // 4)
    out = n * (k + 2) * 4
    for i, size in enumerate(sizes.values()):
        end = (size + 15) // 16 * 16
        for offset, refused in ((0, True), (end - 16, True), (end, False), (-out, False), (16 - out, True)):
            at("out", 4096 * (i + 1) + offset, out // 4)
            call = lambda: rt.verify("target", "draft", "tokens", "u", vocab, n, k, lens="lens", temperature="temp", out="out", blocking=False)
            if refused:
                with pytest.raises(ValueError, match="of their own"):
                    call()
            else:
                call()


def test_a_pitch_that_no_memory_has_is_refused():
    import torch

    from vinf_3080ti_b200.runtime import Runtime

    rt = Runtime()
    room = torch.zeros(64, device="cuda")
    for pitch, n_rows in ((1 << 39, 1 << 30), (1 << 33, (1 << 29) + 1)):
        with pytest.raises(ValueError, match="pitch"):
            rt.bind_i8("w", room.data_ptr(), room.data_ptr(), 16, n_rows, pitch=pitch)
    rt.close()
