// Product of e4m3 activations (a scale for each 128 columns of a row) and e4m3 weights (a scale for each block of 128 x 128):
//   y[t][r] = sum_b sx[b][t] sw[r / 128][b] sum_{k in block b} q[t][k] W[r][k].
// Simple form: a tile of 16 x 16 outputs per block of threads, one output each, on the CUDA cores.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "vqm_kernels.h"

namespace vqm {
namespace {

__device__ __forceinline__ void put(float *y, float v, bool add) { *y = add ? *y + v : v; }
__device__ __forceinline__ void put(__half *y, float v, bool add) { *y = __float2half_rn(add ? __half2float(*y) + v : v); }

template <typename Y>
__global__ void __launch_bounds__(256) qmm_f8_kernel(const QmmF8Args a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ float s_w[16][kF8Block + 1], s_q[16][kF8Block + 1];
    const int x = threadIdx.x & 15, z = threadIdx.x >> 4, row0 = static_cast<int>(blockIdx.x) * 16, n_blocks = (a.cols + kF8Block - 1) / kF8Block;
    const long long tok_pitch = f8_scale_pitch(a.ntok);
    for (long long tok0 = static_cast<long long>(blockIdx.y) * 16; tok0 < a.ntok; tok0 += 16ll * gridDim.y) {
        float acc = 0.0f;
        const int row = row0 + x;
        const long long tok = tok0 + z;
        for (int b = 0; b < n_blocks; ++b) {
            __syncthreads();
            for (int i = threadIdx.x; i < 16 * kF8Block; i += 256) {
                const int r = i / kF8Block, c = i % kF8Block, k = b * kF8Block + c;
                __nv_fp8_e4m3 w, q;
                w.__x = row0 + r < a.rows && k < a.cols ? a.w[(row0 + r) * a.w_pitch + k] : 0;
                q.__x = tok0 + r < a.ntok && k < a.cols ? a.q[(tok0 + r) * f8_pitch(a.cols) + k] : 0;
                s_w[r][c] = static_cast<float>(w);
                s_q[r][c] = static_cast<float>(q);
            }
            __syncthreads();
            float sum = 0.0f;
            for (int c = 0; c < kF8Block; ++c) sum += s_w[x][c] * s_q[z][c];
            if (row < a.rows && tok < a.ntok) acc += sum * (a.q_scales[b * tok_pitch + tok] * a.w_scales[static_cast<size_t>(row / kF8Block) * n_blocks + b]);
        }
        if (row < a.rows && tok < a.ntok) put(static_cast<Y *>(a.y) + tok * a.rows + row, acc, a.add);
    }
}

}  // namespace

cudaError_t launch_qmm_f8(const QmmF8Args &a, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[2];
    const int tok_tiles = (a.ntok + 15) / 16;
    cfg.gridDim = dim3(static_cast<unsigned>((a.rows + 15) / 16), static_cast<unsigned>(tok_tiles < 65535 ? tok_tiles : 65535));
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = launch_attributes(attr, a.overlap, 0);
    return a.y_elem == 2 ? cudaLaunchKernelEx(&cfg, qmm_f8_kernel<__half>, a) : cudaLaunchKernelEx(&cfg, qmm_f8_kernel<float>, a);
}

}  // namespace vqm
