// Product of 8-bit integers:  y[t][r] = sx[t] sw[r] sum_k q[t][k] W[r][k],  sums in 32-bit integers, exact.
#include <cuda_fp16.h>

#include "vqm_kernels.h"

namespace vqm {
namespace {

constexpr int kGroup = 8;  // activation rows that a warp carries along

__global__ void __launch_bounds__(256) qmm_i8_kernel(const QmmI8Args a) {
    const int row = static_cast<int>(blockIdx.x * 8 + (threadIdx.x >> 5)), lane = threadIdx.x & 31;
    if (row >= a.rows) return;
    const int t0 = blockIdx.y * kGroup, m = min(kGroup, a.ntok - t0);
    const long long pitch = i8_pitch(a.cols);
    const int8_t *w = a.w + static_cast<size_t>(row) * a.w_pitch;
    int sum[kGroup] = {};
    for (int c = lane * 4; c < a.cols; c += 128) {
        int word = *reinterpret_cast<const int *>(w + c);
        if (c + 4 > a.cols) word &= (1 << (8 * (a.cols - c))) - 1;  // what lies behind the last column counts nothing
#pragma unroll
        for (int t = 0; t < kGroup; ++t)
            if (t < m) sum[t] = __dp4a(word, *reinterpret_cast<const int *>(a.q + static_cast<size_t>(t0 + t) * pitch + c), sum[t]);
    }
#pragma unroll
    for (int t = 0; t < kGroup; ++t)
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) sum[t] += __shfl_xor_sync(0xffffffffu, sum[t], off);
    if (lane != 0) return;
    for (int t = 0; t < m; ++t) {
        const size_t at = static_cast<size_t>(t0 + t) * a.rows + row;
        const float v = static_cast<float>(sum[t]) * a.q_scales[t0 + t] * a.w_scales[row];
        if (a.y_elem == 2) {
            __half *y = static_cast<__half *>(a.y) + at;
            *y = __float2half_rn(a.add ? __half2float(*y) + v : v);
        } else {
            float *y = static_cast<float *>(a.y) + at;
            *y = a.add ? *y + v : v;
        }
    }
}

}  // namespace

cudaError_t launch_qmm_i8(const QmmI8Args &a, int sm_count, cudaStream_t stream) {
    (void)sm_count;
    const dim3 grid((a.rows + 7) / 8, (a.ntok + kGroup - 1) / kGroup);
    qmm_i8_kernel<<<grid, 256, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace vqm
