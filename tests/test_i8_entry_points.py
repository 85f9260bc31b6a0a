"""CPU checks of the entry points for 8-bit integer passes and verification: refusals before any launch, and the formulas the GPU tests compare with."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from tests import i8_formulas as F
from vinf_3080ti_b200 import _capi


@pytest.fixture(scope="module")
def lib():
    from vinf_3080ti_b200 import build

    build.build()
    return _capi.load()


def test_a_missing_runtime_is_an_error(lib):
    f = ctypes.c_float(1.0)
    for status in (lib.vqm_upload_i8(None, b"w", b"x", 1, ctypes.byref(f), 4, 1, 1), lib.vqm_bind_i8(None, b"w", None, 0, None, 1, 1), lib.vqm_convert_i8(None, b"a", b"b"),
                   lib.vqm_rows_i8(None, b"x", b"q", b"s", 1, 1, 0, None, None, None, None, 0.0), lib.vqm_qmm_i8(None, b"w", b"q", b"s", b"y", 1, 0),
                   lib.vqm_verify(None, b"t", None, None, None, b"u", None, 1, 1, 0, b"o", None)):
        assert status == _capi.ERR_VALUE
        assert b"NULL" in lib.vqm_last_error()


@pytest.mark.parametrize("call", ["upload_i8('w', bytes(1), np.ones(1, 'f'), 1, 1)", "bind_i8('w', 16, 16, 1, 1)", "convert_i8('a', 'b')", "rows_i8('x', 'q', 's', 1)",
                                  "qmm_i8('w', 'q', 's', 'y')", "verify('t', None, None, 'u', 1, 1, 0, out='o')"])
def test_calls_on_a_closed_runtime_are_errors(lib, call):
    from vinf_3080ti_b200.runtime import Runtime

    rt = Runtime.__new__(Runtime)
    rt._lib = lib
    rt._h = ctypes.c_void_p()
    rt.close()
    with pytest.raises(ValueError, match="closed"):
        eval(f"rt.{call}", {"rt": rt, "np": np})


def test_counts_are_checked_before_the_library_is_called(lib):
    from vinf_3080ti_b200.runtime import Runtime

    rt = Runtime.__new__(Runtime)
    rt._lib, rt._h = lib, ctypes.c_void_p()
    for kw in ({"seqs": 0}, {"seqs": -3}, {"drafts": -1}, {"drafts": 256}):
        with pytest.raises(ValueError):
            rt.verify(**{**dict(target="t", draft=None, tokens="k", uniforms="u", vocab=5, seqs=1, drafts=1, out="o"), **kw})
    with pytest.raises(ValueError):
        rt.bind_i8("w", 16, 16, 1, 1, pitch=-1)


def test_the_formulas_on_small_numbers():
    q, s, t = F.rows_i8(np.array([[1.0, -127.0, 0.5, 1.5, 2.5], [0, 0, 0, 0, 0]], np.float32))
    assert q.tolist() == [[1, -127, 0, 2, 2], [0] * 5] and s.tolist() == [1.0, 0.0] and t is None
    q, s, t = F.rows_i8(np.array([[3.0, 0.0]], np.float32), residual=np.array([[1.0, 0.0]], np.float32), norm=np.array([2.0, 1.0], np.float32), eps=0.0)
    assert t.tolist() == [[4.0, 0.0]] and q.tolist() == [[127, 0]] and abs(float(s[0]) - 2 * np.sqrt(2) / 127) < 1e-8
    y, sums = F.qmm_i8(np.array([[1, 2], [-128, 127]], np.int8), np.array([0.5, 2.0], np.float32), np.array([[3, -1]], np.int8), np.array([4.0], np.float32))
    assert sums.tolist() == [[1, -511]] and y.tolist() == [[2.0, -4088.0]]


def test_verification_on_small_numbers():
    logs = np.log(np.array([[0.5, 0.3, 0.2], [0.1, 0.1, 0.8]], np.float64))
    target, draft = logs[None], np.log(np.array([[[0.25, 0.7, 0.05]]]))
    tokens = np.array([[1]])
    # accepted while u 0.7 < 0.3; then the bonus from the second row
    assert F.verify(target, draft, tokens, np.array([[0.42, 0.15]])).tolist() == [[1, 1, 1]]
    assert F.verify(target, draft, tokens, np.array([[0.42, 0.25]])).tolist() == [[1, 1, 2]]
    # refused: the rest is 0.25, 0, 0.15
    assert F.verify(target, draft, tokens, np.array([[0.44, 0.62]])).tolist() == [[0, 0, -1]]
    assert F.verify(target, draft, tokens, np.array([[0.44, 0.63]])).tolist() == [[0, 2, -1]]
    # without the draft's probabilities: accepted while u < 0.3, the rest is 0.5, 0, 0.2
    assert F.verify(target, None, tokens, np.array([[0.29, 0.0]])).tolist() == [[1, 1, 0]]
    assert F.verify(target, None, tokens, np.array([[0.31, 0.75]])).tolist() == [[0, 2, -1]]
    assert F.verify(target, None, tokens, np.array([[0.31, 0.7]])).tolist() == [[0, 0, -1]]


@pytest.mark.parametrize("native", [True, False], ids=["native", "ctypes"])
def test_calls_hand_their_arguments_on(lib, native, monkeypatch):
    got = []
    P, S, I, Fl = ctypes.c_void_p, ctypes.c_char_p, ctypes.c_int, ctypes.c_float

    def fake(*kinds):
        @ctypes.CFUNCTYPE(I, P, *kinds)
        def fn(*args):
            got.append(args)
            return 4

        return fn

    fakes = {"rows_i8": fake(S, S, S, I, I, I, S, S, S, S, Fl), "qmm_i8": fake(S, S, S, S, I, I), "verify": fake(S, S, S, S, S, S, I, I, I, S, P)}
    if native:
        call = {n: lambda *a, n=n: getattr(_capi.pycall(), n)(ctypes.cast(fakes[n], P).value, *a) for n in fakes}
    else:
        monkeypatch.setattr(_capi, "_callers", {})
        monkeypatch.setattr(_capi, "pycall", lambda: None)
        monkeypatch.setattr(_capi, "load", lambda: type("Lib", (), {"vqm_" + n: staticmethod(f) for n, f in fakes.items()}))
        call = {n: _capi.caller(n) for n in fakes}
    host = (ctypes.c_int * 4)()
    at = ctypes.addressof(host)
    assert call["rows_i8"](123, "x", "größe", "s", 5120, np.int64(3), 9, None, "r", None, "g", 0.5) == 4
    assert call["qmm_i8"](123, "w", "q", "s", "y", 2**32 + 9, True) == 4
    assert call["verify"](123, "t", None, "k", None, "u", "temp", 9, 2, 1, "o", at) == 4
    assert call["verify"](123, "t", "d", None, "l", "u", None, 9, 2, 0, "o", 0) == 4
    assert got == [(123, b"x", "größe".encode(), b"s", 5120, 3, 9, None, b"r", None, b"g", 0.5), (123, b"w", b"q", b"s", b"y", 9, 1),
                   (123, b"t", None, b"k", None, b"u", b"temp", 9, 2, 1, b"o", at), (123, b"t", b"d", None, b"l", b"u", None, 9, 2, 0, b"o", None)]
    for name, args in (("rows_i8", (None, "x", "q", "s", 1, 1, 0, None, None, None, None, 0.0)), ("qmm_i8", (None, "w", "q", "s", "y", 1, 0))):
        with pytest.raises((TypeError, ValueError)):  # a closed runtime
            call[name](*args)
    if native:
        for name, args in (("rows_i8", (1, b"x", "q", "s", 1, 1, 0, None, None, None, None, 0.0)), ("rows_i8", (1, "x", "q", "s", 1, 1, 0, None, None, None, 5, 0.0)),
                           ("qmm_i8", (1, "w", None, "s", "y", 1, 0)), ("verify", (1, None, "d", None, "l", "u", None, 9, 2, 0, "o", 0))):
            with pytest.raises(AttributeError):
                call[name](*args)
        for name, args in (("rows_i8", (1, "x", "q", "s", "a", 1, 0, None, None, None, None, 0.0)), ("rows_i8", (1, "x", "q", "s", 1, 1, 0, None, None, None, None, "e")),
                           ("qmm_i8", (1, "w", "q", "s", "y", None, 0)), ("qmm_i8", (1, "w", "q", "s", "y", 1))):
            with pytest.raises((TypeError, ValueError)):
                call[name](*args)
    assert len(got) == 4
