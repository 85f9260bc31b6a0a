"""Whether a launch may overlap the one before it is the caller's to say: the launchers of the newer passes, compiled with a launch that only looks at its attributes."""
from __future__ import annotations

import subprocess

import pytest

from vinf_3080ti_b200 import build

HEAD = """
#include <cuda_runtime.h>
#include <cstdio>
#include <cstring>
static int g_launches = 0, g_overlap = 0, g_clusters = 0;
template <typename... A> static cudaError_t fake_launch(const cudaLaunchConfig_t *cfg, A...) {
    ++g_launches;
    for (unsigned i = 0; i < cfg->numAttrs; ++i) {
        if (cfg->attrs[i].id == cudaLaunchAttributeProgrammaticStreamSerialization) g_overlap += cfg->attrs[i].val.programmaticStreamSerializationAllowed;
        if (cfg->attrs[i].id == cudaLaunchAttributeClusterDimension) ++g_clusters;
    }
    return cudaSuccess;
}
template <typename... A> static cudaError_t fake_room(int *n, A...) { *n = 18; return cudaSuccess; }
template <typename T> static cudaError_t fake_attributes(cudaFuncAttributes *is, T) { std::memset(is, 0, sizeof(*is)); is->numRegs = 255; return cudaSuccess; }
template <typename... A> static cudaError_t fake_set(A...) { return cudaSuccess; }
#define cudaLaunchKernelEx fake_launch
#define cudaOccupancyMaxActiveClusters fake_room
#define cudaFuncGetAttributes fake_attributes
#define cudaFuncSetAttribute fake_set
#include "KERNEL"
static void said(bool overlap) {
    std::printf("%d %d %d %d\\n", overlap ? 1 : 0, g_launches, g_overlap, g_clusters);
    g_launches = g_overlap = g_clusters = 0;
}
"""
ENCODER = """
namespace vqm {
template <typename T> struct Encoded;
template <typename... A> struct Encoded<CUresult (*)(A...)> { static CUresult call(A...) { return CUDA_SUCCESS; } };
cudaError_t tc_encoder(TcEncode *out) { *out = &Encoded<TcEncode>::call; return cudaSuccess; }
}
"""
MAINS = {
    "vqm_logprobs.cu": """
int main() {
    for (bool overlap : {false, true})
        for (int rows : {1, 16, 500})
            for (int elem : {2, 4}) {
                vqm::LogprobsArgs a{};
                a.vocab = 151936, a.rows = rows, a.top = 3, a.elem = elem;
                if (vqm::launch_logprobs(a, overlap, nullptr) != cudaSuccess) return 1;
                said(overlap);
            }
}
""",
    "vqm_rows_f8.cu": """
int main() {
    float g = 0.0f;
    for (bool overlap : {false, true})
        for (int cols : {500, 5120, 5121, 12288, 40000})
            for (bool norm : {false, true}) {
                vqm::RowsF8Args a{};
                a.cols = cols, a.ntok = 700, a.elem = 4, a.norm_w = norm ? &g : nullptr;
                if (vqm::launch_rows_f8(a, overlap, 148, nullptr) != cudaSuccess) return 1;
                said(overlap);
            }
}
""",
    "vqm_qmm_f8.cu": ENCODER + """
int main() {
    for (bool overlap : {false, true})
        for (int rows : {1000, 40000})
            for (int ntok : {1, 20, 50, 100, 600}) {
                vqm::QmmF8Args a{};
                a.rows = rows, a.cols = 5120, a.w_pitch = 5120, a.ntok = ntok, a.y_elem = 4, a.overlap = overlap;
                if (vqm::launch_qmm_f8(a, nullptr) != cudaSuccess) return 1;
                said(overlap);
            }
}
""",
}


@pytest.mark.parametrize("kernel", MAINS)
def test_launches_overlap_if_the_caller_says_so(tmp_path, kernel):
    source, program = tmp_path / "launches.cu", tmp_path / "launches"
    source.write_text(HEAD.replace("KERNEL", kernel) + MAINS[kernel])
    subprocess.run([build._nvcc(), "-O1", "-Xptxas", "-O0", *build.NVCC_FLAGS[:2], "-std=c++17", "-I", str(build.CSRC), str(source), "-o", str(program)], check=True, capture_output=True)
    lines = [tuple(map(int, line.split())) for line in subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout.splitlines()]
    assert len(lines) >= 12 and {line[0] for line in lines} == {0, 1}
    for overlap, launches, overlapping, _ in lines:
        assert launches > 0 and overlapping == overlap * launches
    if kernel != "vqm_rows_f8.cu":
        assert any(line[3] for line in lines)  # some in clusters
