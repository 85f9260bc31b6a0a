"""Whether a launch may overlap the one before it, and its clusters: the attributes that the launchers hand to the driver."""
from __future__ import annotations

import subprocess

import pytest

from vinf_3080ti_b200 import build

MAIN = """
#include "vqm_kernels.h"
#include <cstdio>
int main() {
    for (int overlap = 0; overlap < 2; ++overlap)
        for (int cluster : {0, 1, 4, 16}) {
            cudaLaunchAttribute attr[2];
            const unsigned n = vqm::launch_attributes(attr, overlap != 0, cluster);
            int serial = 0, x = 0;
            for (unsigned i = 0; i < n; ++i) {
                if (attr[i].id == cudaLaunchAttributeProgrammaticStreamSerialization) serial += attr[i].val.programmaticStreamSerializationAllowed;
                else if (attr[i].id == cudaLaunchAttributeClusterDimension && attr[i].val.clusterDim.y == 1 && attr[i].val.clusterDim.z == 1) x += static_cast<int>(attr[i].val.clusterDim.x);
                else return 1;
            }
            std::printf("%d %d %u %d %d\\n", overlap, cluster, n, serial, x);
        }
}
"""


def test_attributes_say_what_was_asked_for(tmp_path):
    source, program = tmp_path / "attributes.cu", tmp_path / "attributes"
    source.write_text(MAIN)
    subprocess.run([build._nvcc(), "-std=c++17", "-I", str(build.CSRC), str(source), "-o", str(program)], check=True)
    lines = subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout.splitlines()
    assert len(lines) == 8
    for overlap, cluster, n, serial, x in (map(int, line.split()) for line in lines):
        assert (n, serial, x) == (overlap + (cluster > 0), overlap, cluster)


@pytest.mark.parametrize("name", ["vqm_gemm.cu", "vqm_gemm_tc5.cu", "vqm_qmm_i8.cu", "vqm_rows_i8.cu", "vqm_verify.cu"])
def test_no_launcher_asks_for_overlap_by_itself(name):
    source = (build.CSRC / name).read_text()
    assert "launch_attributes(" in source and "ProgrammaticStreamSerialization" not in source
