"""Products of 8-bit rows of which a part gives up.  A program built here has the blocks of one part of a tile's columns multiply no more than the first block of
them: their writers' waits, which have a limit, run out, and with them those of whoever waits for their sums.  The launch ends by itself, its status word says so, and launches
behind it are as they would be."""
from __future__ import annotations

import subprocess

import pytest

from vinf_3080ti_b200 import build

pytestmark = pytest.mark.gpu

# Weights, activations and scales of 1 onto outputs of 7: what is right is 7 + cols.  For each size: the launch's error, its status, how many outputs are as they were, how many right, how
# many neither; then those of a launch of one part, whose blocks do not stall.
MAIN = """
#include "KERNEL"
#include <cstdio>
#include <vector>
using namespace vqm;
static void *made(size_t bytes, int value) {
    void *p = nullptr;
    if (cudaMalloc(&p, bytes) != cudaSuccess || cudaMemset(p, value, bytes) != cudaSuccess) return nullptr;
    return p;
}
static float *floats(size_t n, float v) {
    std::vector<float> host(n, v);
    void *p = made(4 * n, 0);
    if (p != nullptr) cudaMemcpy(p, host.data(), 4 * n, cudaMemcpyHostToDevice);
    return static_cast<float *>(p);
}
static int once(int rows, int cols, int ntok, bool add) {
    const size_t pitch = (cols + 15) / 16 * 16, blocks = (cols + 127) / 128, outputs = static_cast<size_t>(rows) * ntok;
    void *w = made(pitch * rows, ONE), *q = made(pitch * ntok, ONE), *status = made(4, 0);
    float *ws = floats((static_cast<size_t>(rows) + 127) * (blocks + 1), 1.0f), *qs = floats(blocks * (ntok + 4), 1.0f), *y = floats(outputs, 7.0f);
    if (w == nullptr || q == nullptr || status == nullptr || ws == nullptr || qs == nullptr || y == nullptr) return 1;
    ARGS a{};
    a.w = static_cast<decltype(a.w)>(w);
    a.q = static_cast<decltype(a.q)>(q);
    a.w_scales = ws, a.q_scales = qs, a.y = y, a.status = static_cast<unsigned *>(status);
    a.w_pitch = static_cast<long long>(pitch);
    a.rows = rows, a.cols = cols, a.ntok = ntok, a.y_elem = 4, a.add = add, a.overlap = true;
    const cudaError_t err = LAUNCH(a, nullptr), done = cudaDeviceSynchronize();
    std::vector<float> out(outputs);
    unsigned code = 99;
    cudaMemcpy(&code, status, 4, cudaMemcpyDeviceToHost);
    cudaMemcpy(out.data(), y, 4 * outputs, cudaMemcpyDeviceToHost);
    size_t same = 0, right = 0;
    for (float v : out) same += v == 7.0f, right += v == (add ? 7.0f : 0.0f) + static_cast<float>(cols);
    std::printf("%d %u %zu %zu %zu\\n", static_cast<int>(err != cudaSuccess ? err : done), code, same, right, outputs - same - right);
    std::fflush(stdout);
    for (void *p : {w, q, status, static_cast<void *>(ws), static_cast<void *>(qs), static_cast<void *>(y)}) cudaFree(p);
    return err != cudaSuccess || done != cudaSuccess;
}
int main(int argc, char **argv) {
    for (int i = 1; i + 3 < argc; i += 4) {
        if (once(std::atoi(argv[i]), std::atoi(argv[i + 1]), std::atoi(argv[i + 2]), argv[i + 3][0] == '1')) return 1;
        if (once(40000, 256, std::atoi(argv[i + 2]), false)) return 1;
    }
    return 0;
}
"""


def results(tmp_path, kernel, stalled, sizes):
    """[(rows, ntok), launch that stalls, launch of one part] for each size; a launch is (error, status, outputs as they were, right, neither)"""
    source, program = tmp_path / "given_up.cu", tmp_path / "given_up"
    one, args, launch = {"vqm_qmm_f8.cu": ("0x38", "QmmF8Args", "launch_qmm_f8"), "vqm_qmm_i8.cu": ("1", "QmmI8Args", "launch_qmm_i8")}[kernel]
    source.write_text("#include <cstdlib>\n" + MAIN.replace("KERNEL", kernel).replace("ONE", one).replace("ARGS", args).replace("LAUNCH", launch))
    subprocess.run([build._nvcc(), *build.NVCC_FLAGS[:5], f"-DVQM_STALLED_PART={stalled}", "-I", str(build.CSRC), str(source), str(build.CSRC / "vqm_tcmv_maps.cu"), "-o", str(program)],
                   check=True, capture_output=True)
    done = subprocess.run([str(program), *[str(v) for size in sizes for v in size]], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stdout + done.stderr
    lines = [tuple(map(int, line.split())) for line in done.stdout.splitlines()]
    assert len(lines) == 2 * len(sizes)
    return [((rows, ntok), lines[2 * i], lines[2 * i + 1]) for i, (rows, _, ntok, _) in enumerate(sizes)]


# few rows with sums in memory of their own and where the stages were, more rows, pairs
F8_SIZES = [(1024, 5120, 4, 1), (1024, 17408, 4, 0), (1000, 5120, 30, 1), (1024, 17408, 50, 1), (1024, 17408, 128, 1), (1001, 17408, 128, 0), (5120, 17408, 256, 1)]


@pytest.fixture(scope="module")
def second_part_stalls(tmp_path_factory):
    return results(tmp_path_factory.mktemp("f8"), "vqm_qmm_f8.cu", 1, F8_SIZES)


def test_a_launch_that_gives_up_ends_and_leaves_the_next_as_it_is(second_part_stalls):
    for (rows, ntok), first, second in second_part_stalls:
        assert first[:2] == (0, 1)
        assert second == (0, 0, 0, 40000 * ntok, 0)


def test_sums_that_a_part_has_given_up_reach_no_output(second_part_stalls):
    """Every output needs that part's: all of them are as they were."""
    for (rows, ntok), first, _ in second_part_stalls:
        assert first == (0, 1, rows * ntok, 0, 0), (rows, ntok)


def test_blocks_that_share_no_columns_write_nothing_once_they_have_given_up(tmp_path):
    for (rows, ntok), first, second in results(tmp_path, "vqm_qmm_f8.cu", 0, [(1024, 5120, 4, 1), (1024, 17408, 128, 1), (5120, 17408, 256, 1)]):
        assert first[:2] == (0, 1)
        assert second == (0, 1, 40000 * ntok, 0, 0)


def test_the_same_of_8_bit_integers(tmp_path):
    for (rows, ntok), first, second in results(tmp_path, "vqm_qmm_i8.cu", 1, [(1024, 5120, 4, 1), (1000, 17408, 50, 1), (1024, 17408, 200, 0), (1024, 17408, 300, 1)]):
        assert first == (0, 1, rows * ntok, 0, 0), (rows, ntok)
        assert second == (0, 0, 0, 40000 * ntok, 0)
