"""Whether two pieces of memory overlap, as the calls that write beside reads ask, against sets of bytes."""
from __future__ import annotations

import random
import subprocess

from vinf_3080ti_b200 import build

MAIN = """
#include "vqm_kernels.h"
#include <cstdio>
#include <cstdlib>
int main(int argc, char **argv) {
    auto number = [&](int i) { return std::strtoull(argv[i], nullptr, 10); };
    for (int i = 1; i + 3 < argc; i += 4)
        std::printf("%d\\n", vqm::overlap({reinterpret_cast<void *>(number(i)), number(i + 1)}, {reinterpret_cast<void *>(number(i + 2)), number(i + 3)}) ? 1 : 0);
}
"""


def test_overlap(tmp_path):
    source, program = tmp_path / "overlap.cu", tmp_path / "overlap"
    source.write_text(MAIN)
    subprocess.run([build._nvcc(), "-std=c++17", "-I", str(build.CSRC), str(source), "-o", str(program)], check=True)
    rng = random.Random(1)
    cases = [(rng.randrange(1, 30), rng.randrange(0, 12), rng.randrange(1, 30), rng.randrange(0, 12)) for _ in range(2000)]
    cases += [(0, 50, 1, 50), (1, 50, 0, 50), (0, 50, 0, 50), (5, 0, 5, 0), (5, 1, 5, 1), (2**47, 2**40, 2**47 + 2**40 - 1, 1), (2**47, 2**40, 2**47 + 2**40, 1), (2**47 + 5, 1, 2**47, 2**40)]
    got = subprocess.run([str(program), *(str(v) for c in cases for v in c)], check=True, capture_output=True, text=True).stdout.split()
    for (p, n, q, m), answer in zip(cases, got, strict=True):
        assert answer == str(int(p != 0 and q != 0 and max(p, q) < min(p + n, q + m))), (p, n, q, m)
