"""The distance from a half within which rows_i8 rounds in 64 bits covers what fp32 may be off by.  Documented errors, in units of 2^-24 (half a step
behind a power of two): a product, a sum, a conversion or __fdiv_rn 1; ex2.approx 2^-22; rcp.approx one step."""
from __future__ import annotations

import subprocess

import numpy as np
import pytest

from vinf_3080ti_b200 import build

UNIT = 2.0**-24
PRODUCT, DIVISION, EX2, RECIPROCAL = 1, 1, 4, 2


@pytest.fixture(scope="module")
def off(tmp_path_factory):
    folder = tmp_path_factory.mktemp("margins")
    source, program = folder / "margins.cu", folder / "margins"
    source.write_text('#include "vqm_kernels.h"\n#include <cstdio>\nint main() { std::printf("%.9g %.9g %.9g\\n", vqm::kI8Off, vqm::kI8GatedOff, vqm::kI8GatedOffPerX); }\n')
    subprocess.run([build._nvcc(), "-std=c++17", "-I", str(build.CSRC), str(source), "-o", str(program)], check=True)
    return [float(v) for v in subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout.split()]


def test_the_margins_cover_the_documented_errors(off):
    plain, gated, per_x = (v / UNIT for v in off)
    rounded = 0.5  # of the bound at 1/2: 2^-26
    # (products of 1 + error: second-order terms are within a millionth)
    assert plain >= (PRODUCT + 1 + DIVISION + PRODUCT + rounded) * 1.000001
    assert gated >= (2 * PRODUCT + DIVISION + PRODUCT + EX2 + 1 + RECIPROCAL + rounded) * 1.000001
    constant = abs(float(np.float32(1.44269504)) * np.log(2.0) - 1.0) / UNIT  # of the argument -x log2(e)
    assert per_x >= (PRODUCT + constant) * 1.000001


@pytest.mark.parametrize("whole", [0, 1, 2, 7, 63, 126])
def test_values_next_to_a_half_are_seen(off, whole):
    """t = (e g) (r / s) in fp32 against 64 bits."""
    f32, rng, n = np.float32, np.random.default_rng(whole), 200_000
    for spread in (4, 4096, 1 << 22):
        def mantissa():
            return 1.0 + rng.integers(0, spread, n) * 2.0**-23

        e, s, r = mantissa(), mantissa(), mantissa() + rng.uniform(-0.49, 0.49, n) * 2.0**-23
        g = f32((whole + 0.5) * s / (r * e)).astype(np.float64)
        want = np.rint(e * g * r / s)
        t = f32(f32(f32(e) * f32(g)) * (f32(r) / f32(s))).astype(np.float64)
        near = np.abs(t - np.rint(t)) > f32(0.5 - np.abs(t) * off[0])
        assert ((np.rint(t) == want) | near).all()
