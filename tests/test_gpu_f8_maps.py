"""How many tensor maps a product of e4m3 rows encodes on the host: those of its operands, and of its outputs only where it writes by them."""
from __future__ import annotations

import subprocess

import pytest

from vinf_3080ti_b200 import build

pytestmark = pytest.mark.gpu

MAIN = """
#include "vqm_qmm_f8.cu"
#define tc_encoder real_encoder
#include "vqm_tcmv_maps.cu"
#undef tc_encoder
#include <cstdio>
#include <cstdlib>
static vqm::TcEncode g_real = nullptr;
static int g_count = 0;
template <typename... A> struct Counted;
template <typename R, typename... A> struct Counted<R (*)(A...)> {
    static R call(A... a) { ++g_count; return g_real(a...); }
};
namespace vqm {
cudaError_t tc_encoder(TcEncode *out) {
    const cudaError_t err = real_encoder(&g_real);
    *out = &Counted<TcEncode>::call;
    return err;
}
}
int main(int argc, char **argv) {
    void *p = nullptr;  // zeros as weights, activations, scales; never outputs
    if (cudaMalloc(&p, 512 << 20) != cudaSuccess || cudaMemset(p, 0, 512 << 20) != cudaSuccess) return 1;
    void *y = nullptr;
    if (cudaMalloc(&y, 64 << 20) != cudaSuccess) return 1;
    for (int i = 1; i + 3 < argc; i += 4) {
        vqm::QmmF8Args a{};
        a.w = a.q = static_cast<uint8_t *>(p);
        a.w_scales = a.q_scales = static_cast<float *>(p);
        a.y = y;
        a.status = static_cast<unsigned *>(y) + (60 << 18);
        a.rows = std::atoi(argv[i]), a.cols = std::atoi(argv[i + 1]), a.ntok = std::atoi(argv[i + 2]), a.add = argv[i + 3][0] == '1';
        a.w_pitch = vqm::f8_pitch(a.cols), a.y_elem = 4;
        g_count = 0;
        if (vqm::launch_qmm_f8(a, nullptr) != cudaSuccess || cudaDeviceSynchronize() != cudaSuccess) return 1;
        std::printf("%d\\n", g_count);
    }
    return 0;
}
"""

# rows, columns, activation rows, whether onto what is there, maps: few rows; columns that are shared, without and in pairs; single blocks; pairs; rows that do not begin on 16 bytes
CALLS = [(17408, 5120, 4, 0, 2), (1024, 17408, 128, 0, 2), (5120, 17408, 256, 0, 2), (17408, 5120, 100, 0, 3), (17408, 5120, 512, 0, 3), (17408, 5120, 100, 1, 2), (17407, 5120, 100, 0, 2)]


def test_outputs_have_a_map_only_where_they_are_written_by_it(tmp_path):
    source, program = tmp_path / "maps.cu", tmp_path / "maps"
    source.write_text(MAIN)
    subprocess.run([build._nvcc(), *build.NVCC_FLAGS[:5], "-I", str(build.CSRC), str(source), "-o", str(program)], check=True, capture_output=True)
    done = subprocess.run([str(program), *[str(v) for call in CALLS for v in call[:4]]], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stdout + done.stderr
    assert [int(line) for line in done.stdout.split()] == [call[4] for call in CALLS]
