// Activation rows in 8-bit floating point (e4m3) with a scale for each 128 columns, after what a layer does to them on the way to a projection:
//   v = x,  or silu(x) * x2,  or h = x + residual (rounded to its type and stored);   n = v * g / sqrt(mean(v^2) + eps), or v;
//   s = max |n| / 448 over 128 columns, in fp32,   q = n / s (in fp32) rounded to the nearest e4m3 value, ties to even.
// Simple form: a block of threads per row, every pass reads the row again.
#include <cuda_fp16.h>

#include "vqm_kernels.h"

namespace vqm {
namespace {

constexpr float kMost = 448.0f;  // of e4m3

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ void put(float *p, float v) { *p = v; }
__device__ __forceinline__ void put(__half *p, float v) { *p = __float2half_rn(v); }

// silu(x) * x2.  With h = exp(-|x| / 2) neither a far negative x, whose silu is exp(x) x, nor a large x2 leaves fp32 on the way.
__device__ __forceinline__ float gated(float x, float x2) {
    const float h = expf(-0.5f * fabsf(x)), g = x < 0.0f ? h : 1.0f;
    return x * g / (1.0f + h * h) * (x2 * g);
}

// Two values as e4m3, the first in the lower byte; what is beyond 448 becomes that.
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    uint16_t out;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(out) : "f"(b), "f"(a));
    return out;
}

template <typename T>
__global__ void __launch_bounds__(256) rows_f8_kernel(const RowsF8Args a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ double s_sum[8];
    const size_t at = static_cast<size_t>(blockIdx.x) * a.cols;
    const T *x = static_cast<const T *>(a.x) + at, *x2 = static_cast<const T *>(a.x2) + at, *res = static_cast<const T *>(a.residual) + at;
    T *total = static_cast<T *>(a.total) + at;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    double sum = 0.0;
    for (int c = threadIdx.x; c < a.cols; c += 256) {
        float v = as_float(x[c]);
        if (a.residual != nullptr) {
            put(total + c, v + as_float(res[c]));
            v = as_float(total[c]);
        } else if (a.x2 != nullptr) {
            v = gated(v, as_float(x2[c]));
        }
        sum += static_cast<double>(v) * v;
    }
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    sum = 0.0;
    for (int w = 0; w < 8; ++w) sum += s_sum[w];
    const double factor = 1.0 / sqrt(sum / a.cols + a.eps);
    // a warp per 128 columns
    uint8_t *q = a.q + static_cast<size_t>(blockIdx.x) * f8_pitch(a.cols);
    for (int b = warp; b * kF8Block < a.cols; b += 8) {
        float n[4];
        uint32_t most = 0;
        for (int i = 0; i < 4; ++i) {
            const int c = b * kF8Block + lane * 4 + i;
            n[i] = 0.0f;
            if (c >= a.cols) continue;
            float v = a.residual != nullptr ? as_float(total[c]) : as_float(x[c]);
            if (a.x2 != nullptr) v = gated(v, as_float(x2[c]));
            n[i] = a.norm_w != nullptr ? static_cast<float>(v * factor * a.norm_w[c]) : v;
            most = max(most, __float_as_uint(n[i]) & 0x7FFFFFFFu);
        }
        most = __reduce_max_sync(0xFFFFFFFFu, most);
        const bool fine = most < 0x7F800000u;
        const float scale = fine ? __uint_as_float(most) / kMost : __uint_as_float(0x7FFFFFFFu);
        if (lane == 0) a.scales[static_cast<size_t>(b) * f8_scale_pitch(a.ntok) + blockIdx.x] = scale;
        const bool some = fine && scale > 0.0f;
        const uint32_t packed = some ? pack2(n[0] / scale, n[1] / scale) | pack2(n[2] / scale, n[3] / scale) << 16 : 0u;
        if (b * kF8Block + lane * 4 < f8_pitch(a.cols)) *reinterpret_cast<uint32_t *>(q + b * kF8Block + lane * 4) = packed;
    }
}

// A block of 128 x 128 weights by 256 threads.
__global__ void __launch_bounds__(256) blocks_f8_kernel(const float *w, uint8_t *q, float *scales, int rows, int cols) {
    __shared__ uint32_t s_most;
    const int row0 = static_cast<int>(blockIdx.y) * kF8Block, col0 = static_cast<int>(blockIdx.x) * kF8Block;
    const int n_rows = min(kF8Block, rows - row0), pitch = static_cast<int>(f8_pitch(cols));
    if (threadIdx.x == 0) s_most = 0;
    __syncthreads();
    const int quad = (threadIdx.x & 31) * 4;  // four columns
    auto value = [&](int r, int i) { return col0 + quad + i < cols ? w[static_cast<size_t>(row0 + r) * cols + col0 + quad + i] : 0.0f; };
    uint32_t most = 0;
    for (int r = threadIdx.x >> 5; r < n_rows; r += 8)
        for (int i = 0; i < 4; ++i) most = max(most, __float_as_uint(value(r, i)) & 0x7FFFFFFFu);
    atomicMax(&s_most, most);
    __syncthreads();
    const bool fine = s_most < 0x7F800000u;
    const float scale = fine ? __uint_as_float(s_most) / kMost : __uint_as_float(0x7FFFFFFFu);
    if (threadIdx.x == 0) scales[static_cast<size_t>(blockIdx.y) * gridDim.x + blockIdx.x] = scale;
    if (col0 + quad >= pitch) return;
    const bool some = fine && scale > 0.0f;
    for (int r = threadIdx.x >> 5; r < n_rows; r += 8)
        *reinterpret_cast<uint32_t *>(q + static_cast<size_t>(row0 + r) * pitch + col0 + quad) =
            some ? pack2(value(r, 0) / scale, value(r, 1) / scale) | pack2(value(r, 2) / scale, value(r, 3) / scale) << 16 : 0u;
}

}  // namespace

cudaError_t launch_rows_f8(const RowsF8Args &a, bool overlap, int sm_count, cudaStream_t stream) {
    (void)sm_count;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[2];
    cfg.gridDim = dim3(static_cast<unsigned>(a.ntok));
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = launch_attributes(attr, overlap, 0);
    return a.elem == 2 ? cudaLaunchKernelEx(&cfg, rows_f8_kernel<__half>, a) : cudaLaunchKernelEx(&cfg, rows_f8_kernel<float>, a);
}

cudaError_t launch_blocks_f8(const float *w, uint8_t *q, float *scales, int rows, int cols, cudaStream_t stream) {
    // (a tensor's rows come in parts of 65535 blocks at most)
    for (int r = 0; r < rows; r += 65535 * kF8Block) {
        const int n = rows - r < 65535 * kF8Block ? rows - r : 65535 * kF8Block;
        blocks_f8_kernel<<<dim3(static_cast<unsigned>(f8_blocks(cols)), static_cast<unsigned>(f8_blocks(n))), 256, 0, stream>>>(
            w + static_cast<size_t>(r) * cols, q + static_cast<size_t>(r) * f8_pitch(cols), scales + static_cast<size_t>(r / kF8Block) * f8_blocks(cols), n, cols);
        if (const cudaError_t err = cudaGetLastError(); err != cudaSuccess) return err;
    }
    return cudaSuccess;
}

}  // namespace vqm
