"""Memory that is written while other blocks still read it: calls of passes in 8-bit floating point and of log probabilities refuse it whatever names it goes by.  What only touches
is not refused."""
from __future__ import annotations

import numpy as np
import pytest

from tests import f8_formulas as F

pytestmark = pytest.mark.gpu

COLS, NTOK, ROWS = 136, 3, 20
PAGE = 8192


@pytest.fixture()
def memory():
    """A runtime and a function that binds names at offsets of one piece of memory."""
    import torch

    from vinf_3080ti_b200.runtime import Runtime

    rt = Runtime()
    room = torch.zeros(32 * PAGE, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()

    def at(name, offset, n, elem=4):
        rt.bind(name, room.data_ptr() + offset, n, elem)

    yield rt, at, room
    rt.synchronize()
    rt.close()


def around(length, size):
    """Where `size` bytes may lie about `length` that begin at 0, and whether they meet."""
    end = (length + 15) // 16 * 16
    return ((0, True), (end - 16, True), (end, False), (-((size + 15) // 16 * 16), False), (16 - (size + 15) // 16 * 16, True))


def refused_or_not(call, refused):
    if refused:
        with pytest.raises(ValueError, match="of their own"):
            call()
    else:
        call()


ROW_SIZES = {"x": NTOK * COLS * 4, "r": NTOK * COLS * 4, "t": NTOK * COLS * 4, "g": COLS * 4, "h": NTOK * COLS * 2, "hr": NTOK * COLS * 2}
Q, S = NTOK * F.pitch(COLS), F.blocks(COLS) * F.scale_pitch(NTOK)


@pytest.mark.parametrize("kw", [{}, {"norm": "g"}, {"residual": "r"}, {"residual": "r", "total": "x"}, {"residual": "r", "total": "t"}, {"residual": "x"}, {"silu_mul": "r"}, {"silu_mul": "x"},
                                {"x": "h"}, {"x": "h", "residual": "hr", "total": "h"}], ids=str)
def test_rows(memory, kw):
    rt, at, _ = memory
    for i, (name, size) in enumerate(ROW_SIZES.items()):
        elem = 2 if name.startswith("h") else 4
        at(name, PAGE * (i + 1), size // elem, elem)
    at("q", PAGE * 10, Q, 1)
    at("s", PAGE * 11, S)

    def call(**more):
        a = {"x": "x", "q": "q", "scales": "s", "cols": COLS, "ntok": NTOK, **kw, **more}
        rt.rows_f8(a.pop("x"), a.pop("q"), a.pop("scales"), a.pop("cols"), a.pop("ntok"), **a)

    call()
    read = {kw.get("x", "x"), kw.get("residual"), kw.get("total"), kw.get("silu_mul"), kw.get("norm")} - {None}
    for name in read:
        begin = PAGE * (list(ROW_SIZES).index(name) + 1)
        for offset, refused in around(ROW_SIZES[name], Q):
            at("q2", begin + offset, Q, 1)
            refused_or_not(lambda: call(q="q2"), refused)
        for offset, refused in around(ROW_SIZES[name], 4 * S):
            at("s2", begin + offset, S)
            refused_or_not(lambda: call(scales="s2"), refused)
    at("s2", PAGE * 10 + 16, S)
    refused_or_not(lambda: call(scales="s2"), True)  # the scales among the 8-bit rows
    if kw.get("residual") == "r":
        size = ROW_SIZES["x"]
        for name in ("x", "r"):
            begin = PAGE * (list(ROW_SIZES).index(name) + 1)
            for offset, refused in ((0, False), (16, True), (-16, True), (size - 16, True), (size, False), (-size, False)):
                at("t2", begin + offset, NTOK * COLS)
                refused_or_not(lambda: call(total="t2"), refused)


def test_products(memory):
    rt, at, room = memory
    pitch = 144
    rt.bind_f8("w", room.data_ptr() + PAGE, room.data_ptr() + PAGE * 2, COLS, ROWS, pitch=160)
    at("q", PAGE * 3, NTOK * pitch, 1)
    at("s", PAGE * 4, S)
    at("y", PAGE * 5, NTOK * ROWS)
    for add in (False, True):
        rt.qmm_f8("w", "q", "s", "y", NTOK, add=add)
        for page, length in ((3, NTOK * pitch), (4, 4 * S), (1, 160 * (ROWS - 1) + COLS), (2, 4 * F.blocks(COLS))):
            for offset, refused in around(length, NTOK * ROWS * 4):
                at("y2", PAGE * page + offset, NTOK * ROWS)
                refused_or_not(lambda: rt.qmm_f8("w", "q", "s", "y2", NTOK, add=add), refused)


def test_log_probabilities(memory):
    rt, at, _ = memory
    rows, vocab, top = 3, 50, 4
    read = {"logits": rows * vocab * 4, "tokens": rows * 4, "temp": rows * 4}
    written = {"out": rows, "entropy": rows, "top_ids": rows * top, "top_out": rows * top}
    for i, (name, size) in enumerate([*read.items(), *((n, 4 * c) for n, c in written.items())]):
        at(name, PAGE * (i + 1), size // 4)
    where = {name: PAGE * (i + 1) for i, name in enumerate([*read, *written])}

    def call(**more):
        a = {"out": "out", "entropy": "entropy", "top": top, "top_ids": "top_ids", "top_out": "top_out", "temperature": "temp", **more}
        rt.logprobs("logits", "tokens", vocab, rows, **a)

    call()
    for name, count in written.items():
        for other, size in [*read.items(), *((n, 4 * c) for n, c in written.items())]:
            if other == name:
                continue
            for offset, refused in around(size, 4 * count):
                at("moved", where[other] + offset, count)
                refused_or_not(lambda: call(**{name: "moved"}), refused)


def test_a_pitch_that_no_memory_has_is_refused():
    import torch

    from vinf_3080ti_b200.runtime import Runtime

    rt = Runtime()
    room = torch.zeros(64, device="cuda")
    for pitch, n_rows in ((1 << 39, 1 << 30), (1 << 33, (1 << 29) + 1)):
        with pytest.raises(ValueError, match="pitch"):
            rt.bind_f8("w", room.data_ptr(), room.data_ptr(), 16, n_rows, pitch=pitch)
    rt.close()


@pytest.mark.parametrize("kind", ["rows", "product", "logprobs"])
def test_more_elements_than_32_bits_count(kind):
    """Buffers of more than 2^31 elements: the first and the last rows are what they are in a short call."""
    import torch

    from vinf_3080ti_b200.runtime import Runtime

    rt = Runtime()
    gen = torch.Generator(device="cuda").manual_seed(1)

    def bind(name, t):
        rt.bind(name, t.data_ptr(), t.numel(), t.element_size())
        return t

    if kind == "rows":
        cols, n = 5120, 430001
        x = bind("x", torch.randn((n, cols), generator=gen, device="cuda", dtype=torch.float16))
        q, s = bind("q", torch.zeros((n, cols), dtype=torch.int8, device="cuda")), bind("s", torch.zeros((40, F.scale_pitch(n)), device="cuda"))
        gain = bind("g", torch.ones(cols, device="cuda"))
        for norm in (None, "g"):
            torch.cuda.synchronize()
            rt.rows_f8("x", "q", "s", cols, n, norm=norm)
            rt.synchronize()
            some = torch.cat([torch.arange(40), torch.arange(n - 61, n)]).cuda()
            short = bind("x2", x[some].contiguous())
            q2, s2 = bind("q2", torch.zeros((len(some), cols), dtype=torch.int8, device="cuda")), bind("s2", torch.zeros((40, F.scale_pitch(len(some))), device="cuda"))
            torch.cuda.synchronize()
            rt.rows_f8("x2", "q2", "s2", cols, len(some), norm=norm)
            rt.synchronize()
            assert torch.equal(q[some], q2) and torch.equal(s[:, some], s2[:, :len(some)])
        del short, gain
    elif kind == "product":
        cols, rows, n = 128, 151936, 14500
        w, ws = torch.randint(0, 0x40, (rows, cols), generator=gen, device="cuda", dtype=torch.int8), torch.ones((rows // 128, 1), device="cuda")
        rt.bind_f8("w", w.data_ptr(), ws.data_ptr(), cols, rows)
        q, s = bind("q", torch.randint(0, 0x40, (n, cols), generator=gen, device="cuda", dtype=torch.int8)), bind("s", torch.ones((1, n), device="cuda"))
        y = bind("y", torch.zeros((n, rows), dtype=torch.float16, device="cuda"))
        some = torch.cat([torch.arange(40), torch.arange(n - 20, n)]).cuda()
        y2 = bind("y2", torch.zeros((60, rows), dtype=torch.float16, device="cuda"))
        q2, s2 = bind("q2", q[some].contiguous()), bind("s2", s[:, :60].contiguous())
        torch.cuda.synchronize()
        rt.qmm_f8("w", "q2", "s2", "y2", 60)
        for add in (False, True):  # (onto what is there: outputs that do not go out as tiles)
            rt.qmm_f8("w", "q", "s", "y", n, add=add)
            rt.synchronize()
            want = y2 * 2 if add else y2
            # (a block's sum may be added up in another order: a rounding of fp32, which shows in fp16 as one step at most)
            assert ((y[some].float() - want.float()).abs() <= want.float().abs() * 2.0**-9).all() and float(want.float().abs().sum()) > 0
        del q2, s2
    else:
        vocab, n = 151936, 14500
        logits = bind("l", torch.randn((n, vocab), generator=gen, device="cuda", dtype=torch.float16))
        tokens = bind("t", torch.arange(n, device="cuda", dtype=torch.int32))
        out, ids = bind("o", torch.zeros(n, device="cuda")), bind("i", torch.zeros((n, 3), dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        rt.logprobs("l", "t", vocab, n, out="o", top=3, top_ids="i")
        rt.synchronize()
        for r in (0, 1, n - 2, n - 1):
            row = logits[r].double()
            assert abs(float(out[r]) - float(row[int(tokens[r])] - row.logsumexp(0))) < 1e-4
            assert ids[r].tolist() == torch.argsort(row, descending=True, stable=True)[:3].tolist()
    rt.close()
