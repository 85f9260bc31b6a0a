"""The bound within which a draft's test is not left to fp32 sums, against such sums done in numpy."""
from __future__ import annotations

import subprocess

import numpy as np
import pytest

from vinf_3080ti_b200 import build

PARTS = [1, 40, 300, 1000, 3000, 10000, 32768]


@pytest.fixture(scope="module")
def band(tmp_path_factory):
    folder = tmp_path_factory.mktemp("band")
    source, program = folder / "band.cu", folder / "band"
    source.write_text('#include "vqm_kernels.h"\n#include <cstdio>\n#include <cstdlib>\n'
                      "int main(int argc, char **argv) { for (int i = 1; i < argc; ++i) std::printf(\"%.9g\\n\", vqm::verify_band(std::atoll(argv[i]))); }\n")
    subprocess.run([build._nvcc(), "-std=c++17", "-I", str(build.CSRC), str(source), "-o", str(program)], check=True)
    wanted = [*PARTS, 32769, 1 << 40]
    lines = subprocess.run([str(program), *map(str, wanted)], check=True, capture_output=True, text=True).stdout.split()
    return dict(zip(wanted, map(float, lines)))


def test_equal_parts_whose_roundings_go_the_same_way(band):
    parts = np.random.default_rng(1).uniform(4.0, 16.0, 4000).astype(np.float32)
    total = np.zeros_like(parts)
    for n in range(1, PARTS[-1] + 1):
        total += parts
        if n in PARTS:
            off = np.abs(total / (n * parts.astype(np.float64)) - 1.0).max()
            assert 2 * off <= band[n], n  # (one sum too large, the other too small)


def test_sums_that_are_scaled_at_every_part(band):
    """Each part has a new largest: the sum is multiplied by a factor that is off by 2^-22, always to the same side, and rounded twice."""
    rng = np.random.default_rng(2)
    parts = rng.uniform(4.0, 16.0, 300).astype(np.float32)
    factor = np.exp(-rng.uniform(0, 3e-5, 300))  # (a sum stays worth something for all 32768 parts)
    off_factor = (factor * (1.0 + 2.0**-22)).astype(np.float32)
    total, want = np.zeros_like(parts), np.zeros(300)
    for n in range(1, PARTS[-1] + 1):
        total = total * off_factor + parts
        want = want * factor + parts
        if n in PARTS:
            assert 2 * np.abs(total / want - 1.0).max() <= band[n], n


def test_what_a_vocabulary_of_today_costs(band):
    assert band[300] < 4e-4  # drafts in ten thousand that are summed again
    assert band[32769] == band[1 << 40] == 2.0
