"""CPU checks of the entry points for passes in 8-bit floating point and for log probabilities: refusals before any launch, and the formulas the GPU tests compare with."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from tests import f8_formulas as F
from vinf_3080ti_b200 import _capi


@pytest.fixture(scope="module")
def lib():
    from vinf_3080ti_b200 import build

    build.build()
    return _capi.load()


def test_a_missing_runtime_is_an_error(lib):
    f = ctypes.c_float(1.0)
    for status in (lib.vqm_upload_f8(None, b"w", b"x", 1, ctypes.byref(f), 4, 1, 1), lib.vqm_bind_f8(None, b"w", None, 0, None, 1, 1), lib.vqm_convert_f8(None, b"a", b"b"),
                   lib.vqm_rows_f8(None, b"x", b"q", b"s", 1, 1, 0, None, None, None, None, 0.0), lib.vqm_qmm_f8(None, b"w", b"q", b"s", b"y", 1, 0),
                   lib.vqm_logprobs(None, b"l", b"t", None, 1, 1, 0, b"o", None, None, None)):
        assert status == _capi.ERR_VALUE
        assert b"NULL" in lib.vqm_last_error()


@pytest.mark.parametrize("call", ["upload_f8('w', bytes(1), np.ones(1, 'f'), 1, 1)", "bind_f8('w', 16, 16, 1, 1)", "convert_f8('a', 'b')", "rows_f8('x', 'q', 's', 1)",
                                  "qmm_f8('w', 'q', 's', 'y')", "logprobs('l', 't', 5, out='o')"])
def test_calls_on_a_closed_runtime_are_errors(lib, call):
    from vinf_3080ti_b200.runtime import Runtime

    rt = Runtime.__new__(Runtime)
    rt._lib = lib
    rt._h = ctypes.c_void_p()
    rt.close()
    with pytest.raises(ValueError, match="closed"):
        eval(f"rt.{call}", {"rt": rt, "np": np})


def test_a_negative_pitch_is_refused(lib):
    from vinf_3080ti_b200.runtime import Runtime

    rt = Runtime.__new__(Runtime)
    rt._lib, rt._h = lib, ctypes.c_void_p()
    with pytest.raises(ValueError):
        rt.bind_f8("w", 16, 16, 1, 1, pitch=-1)


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

    fakes = {"rows_f8": fake(S, S, S, I, I, I, S, S, S, S, Fl), "qmm_f8": fake(S, S, S, S, I, I), "logprobs": fake(S, S, S, I, I, I, S, S, S, S)}
    if native:
        call = {n: lambda *a, n=n: getattr(_capi.pycall(), n)(ctypes.cast(fakes[n], P).value, *a) for n in fakes}
    else:
        monkeypatch.setattr(_capi, "_callers", {})
        monkeypatch.setattr(_capi, "pycall", lambda: None)
        monkeypatch.setattr(_capi, "load", lambda: type("Lib", (), {"vqm_" + n: staticmethod(f) for n, f in fakes.items()}))
        call = {n: _capi.caller(n) for n in fakes}
    assert call["rows_f8"](123, "x", "größe", "s", 5120, np.int64(3), 9, None, "r", None, "g", 0.5) == 4
    assert call["qmm_f8"](123, "w", "q", "s", "y", 2**32 + 9, True) == 4
    assert call["logprobs"](123, "l", "t", None, 9, 2, 1, "o", None, "i", None) == 4
    assert call["logprobs"](123, "l", "t", "temp", 9, np.int32(2), 0, "größe", "e", None, "v") == 4
    assert got == [(123, b"x", "größe".encode(), b"s", 5120, 3, 9, None, b"r", None, b"g", 0.5), (123, b"w", b"q", b"s", b"y", 9, 1),
                   (123, b"l", b"t", None, 9, 2, 1, b"o", None, b"i", None), (123, b"l", b"t", b"temp", 9, 2, 0, "größe".encode(), b"e", None, b"v")]
    with pytest.raises((TypeError, ValueError)):  # a closed runtime
        call["logprobs"](None, "l", "t", None, 9, 2, 1, "o", None, "i", None)
    if native:
        for args in ((1, None, "t", None, 9, 2, 1, "o", None, "i", None), (1, "l", "t", 5, 9, 2, 1, "o", None, "i", None), (1, "l", "t", None, 9, 2, 1, None, None, "i", None)):
            with pytest.raises(AttributeError):
                call["logprobs"](*args)
        for args in ((1, "l", "t", None, "a", 2, 1, "o", None, "i", None), (1, "l", "t", None, 9, 2, 1, "o", None, "i")):
            with pytest.raises((TypeError, ValueError)):
                call["logprobs"](*args)
    assert len(got) == 4


def test_e4m3_values_are_those_of_another_implementation():
    import torch

    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(codes, F.CODES, equal_nan=True)
    rng = np.random.default_rng(0)
    t = np.concatenate([rng.standard_normal(4000) * 100, rng.standard_normal(4000) * 0.01, F.CODES[:127], (F.CODES[:126] + F.CODES[1:127]) / 2]).astype(np.float32)
    t = t[np.abs(t) <= 448]
    want = torch.from_numpy(t).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(F.encode(t), want) and np.array_equal(F.encode(-t)[t > 0], (want ^ 128)[t > 0])
    assert F.encode(np.array([1e9, -1e9])).tolist() == [0x7E, 0xFE]
    assert F.step(np.array([448.0, 256.0, 255.0, 1.0, 0.99, 2.0**-6, 2.0**-9, 0.0])).tolist() == [32, 32, 16, 0.125, 0.0625, 2.0**-9, 2.0**-9, 2.0**-9]


def test_the_formulas_on_small_numbers():
    n, total = F.values(np.array([[3.0, 0.0]], np.float32), residual=np.array([[1.0, 0.0]], np.float32), norm=np.array([2.0, 1.0], np.float32), eps=0.0)
    assert total.tolist() == [[4.0, 0.0]] and np.allclose(n, [[2 * np.sqrt(2), 0]], rtol=1e-15)
    s = F.scales_of(np.concatenate([np.full((1, 128), -448.0), [[1.0, np.inf]]], 1))
    assert s[0, 0] == 1.0 and np.isnan(s[1, 0])
    one, two = F.encode(1.0), F.encode(-2.0)
    y, most = F.qmm(np.full((129, 130), one), np.array([[1.0, 10.0], [100.0, 1000.0]]), np.full((1, 130), two), np.array([[0.5], [4.0]]))
    assert y[0, 0] == -(128 * 2 * 0.5 + 2 * 2 * 40) and y[0, 128] == 100 * y[0, 0] and np.array_equal(most, -y)


def test_log_probabilities_on_small_numbers():
    x = np.log(np.array([[0.5, 0.25, 0.25], [0.5, 0.25, 0.25]]))
    out, entropy, ids, best = F.logprobs(x, [1, 7], top=4, temperature=[1.0, 0.0])
    assert np.allclose(out, [np.log(0.25), -np.inf]) and np.allclose(entropy, [1.5 * np.log(2), 0])
    assert ids.tolist() == [[0, 1, 2, -1]] * 2
    assert np.allclose(best, [[np.log(0.5), np.log(0.25), np.log(0.25), -np.inf], [0, -np.inf, -np.inf, -np.inf]])
    out, entropy, ids, best = F.logprobs(np.array([[np.nan, -np.inf, -np.inf], [np.inf, 1, np.inf], [-np.inf, 2, 5]]), [0, 0, 1], top=2, temperature=[1, 1, 1e31])
    assert out[0] == -np.inf and entropy[0] == 0 and ids[0].tolist() == [-1, -1]
    assert out[1] == np.log(0.5) and ids[1].tolist() == [0, 2]
    assert out[2] == np.log(0.5) and ids[2].tolist() == [2, 1]
