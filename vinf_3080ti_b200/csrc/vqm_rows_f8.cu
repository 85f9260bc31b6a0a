// Activation rows in 8-bit floating point (e4m3) with a scale for each 128 columns, after what a layer does to them on the way to a projection:
//   v = x,  or silu(x) * x2,  or h = x + residual (rounded to its type and stored);   n = v * g / sqrt(mean(v^2) + eps), or v;
//   s = max |n| / 448 over 128 columns, in fp32,   q = n / s (in fp32) rounded to the nearest e4m3 value, ties to even.
#include <cuda_fp16.h>

#include "vqm_kernels.h"

namespace vqm {
namespace {

constexpr float kMost = 448.0f;  // of e4m3

// silu(x) * x2.  With h = exp(-|x| / 2) neither a far negative x, whose silu is exp(x) x, nor a large x2 leaves fp32 on the way.  h = 2^t (1 + d), where t is the
// argument in fp32 and d what its rounding has left, times ln 2.
__device__ __forceinline__ float gated(float x, float x2) {
    constexpr float kHalfLog2e = 0.72134752044448170f, kRest = static_cast<float>(0.72134752044448170368 - static_cast<double>(kHalfLog2e)), kLn2 = 0.69314718055994531f;
    const float y = -fabsf(x), t = y * kHalfLog2e, d = fmaf(y, kRest, fmaf(y, kHalfLog2e, -t));
    float h, r;
    asm("ex2.approx.f32 %0, %1;" : "=f"(h) : "f"(t));
    h = x == x && y >= -400.0f ? fmaf(h, d * kLn2, h) : x == x ? 0.0f : x;
    const float g = x < 0.0f ? h : 1.0f;
    asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(fmaf(h, h, 1.0f)));
    return x * g * r * (x2 * g);
}

// Two values as e4m3, the first in the lower byte; what is beyond 448 becomes that.
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    uint16_t out;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(out) : "f"(b), "f"(a));
    return out;
}

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float rounded(float v, const float *) { return v; }
__device__ __forceinline__ __half rounded(float v, const __half *) { return __float2half_rn(v); }

// Eight columns from `c` on, zeros from the last on; vec: rows begin on 16 bytes.
__device__ __forceinline__ void load8(const float *p, int left, bool vec, float (&v)[8]) {
    if (vec && left >= 8) {
        const float4 x = *reinterpret_cast<const float4 *>(p), y = *reinterpret_cast<const float4 *>(p + 4);
        v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < left ? p[e] : 0.0f;
    }
}
__device__ __forceinline__ void load8(const __half *p, int left, bool vec, float (&v)[8]) {
    if (vec && left >= 8) {
        const uint4 w = *reinterpret_cast<const uint4 *>(p);
        const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&r[e]));
            v[2 * e] = f.x, v[2 * e + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < left ? __half2float(p[e]) : 0.0f;
    }
}
// Rounds the values to the buffer's type, and stores them.
__device__ __forceinline__ void store8(float *p, int left, bool vec, const float (&v)[8]) {
    if (vec && left >= 8) {
        *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4 *>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < left) p[e] = v[e];
    }
}
__device__ __forceinline__ void store8(__half *p, int left, bool vec, float (&v)[8]) {
    uint32_t r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const __half2 h = __floats2half2_rn(v[2 * e], v[2 * e + 1]);
        r[e] = *reinterpret_cast<const uint32_t *>(&h);
        const float2 f = __half22float2(h);
        v[2 * e] = f.x, v[2 * e + 1] = f.y;
    }
    if (vec && left >= 8) {
        *reinterpret_cast<uint4 *>(p) = make_uint4(r[0], r[1], r[2], r[3]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < left) p[e] = __ushort_as_half(static_cast<unsigned short>(r[e / 2] >> (16 * (e & 1))));
    }
}

// The values of eight columns of a row from c on, before the norm, zeros behind the last; the sums are stored.  By all lanes of a warp, of which 16 side by side have 128 columns;
// c < 0: none.  Rows that do not begin on 16 bytes are read (and sums written) 16 columns after 16 columns, and turned in shared memory.
constexpr int kTurn = 128 + 16;  // floats of 16 lanes (half a warp's banks apart)
template <typename T, bool VEC>
__device__ __forceinline__ void values8(const RowsF8Args &a, size_t row, int c, float *room, float (&v)[8]) {
    if constexpr (VEC) {
        const size_t at = row * a.cols + c;
        const int left = c < 0 ? 0 : a.cols - c;
        if (left <= 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = 0.0f;
            return;
        }
        load8(static_cast<const T *>(a.x) + at, left, true, v);
        if (a.residual != nullptr) {
            float r[8];
            load8(static_cast<const T *>(a.residual) + at, left, true, r);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += r[e];
            store8(static_cast<T *>(a.total) + at, left, true, v);
        } else if (a.x2 != nullptr) {
            float x2[8];
            load8(static_cast<const T *>(a.x2) + at, left, true, x2);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = gated(v[e], x2[e]);
        }
    } else {
        const int lane16 = static_cast<int>(threadIdx.x & 15), c0 = (c < 0 ? a.cols : c - lane16 * 8) + lane16;
        const size_t at = row * a.cols + c0;
        float *const turn = room + threadIdx.x / 16 * kTurn;
        float more[8] = {};
        const T *second = static_cast<const T *>(a.residual != nullptr ? a.residual : a.x2);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c0 + e * 16 < a.cols ? as_float(static_cast<const T *>(a.x)[at + e * 16]) : 0.0f;
        if (second != nullptr)
#pragma unroll
            for (int e = 0; e < 8; ++e) more[e] = c0 + e * 16 < a.cols ? as_float(second[at + e * 16]) : 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (a.residual != nullptr) {
                const T total = rounded(v[e] + more[e], static_cast<const T *>(nullptr));
                if (c0 + e * 16 < a.cols) static_cast<T *>(a.total)[at + e * 16] = total;
                v[e] = as_float(total);
            } else if (a.x2 != nullptr) {
                v[e] = gated(v[e], more[e]);
            }
            turn[lane16 + e * 16] = v[e];
        }
        __syncwarp();
        const float4 p = *reinterpret_cast<const float4 *>(turn + lane16 * 8), q = *reinterpret_cast<const float4 *>(turn + lane16 * 8 + 4);
        __syncwarp();
        v[0] = p.x, v[1] = p.y, v[2] = p.z, v[3] = p.w, v[4] = q.x, v[5] = q.y, v[6] = q.z, v[7] = q.w;
    }
}
// v / scale as fp32 rounds it.  With y = 1 / scale rounded, q = v y and the remainder v - q scale (which one fused multiply and add gives exactly), q + remainder y rounds
// to that (P. Markstein, IBM J. Res. Dev. 34, 1990) wherever nothing of it underflows: for q of 2^-10 on, and smaller ones are nothing in e4m3, where scale is in [2^-80, 2^100].
__device__ __forceinline__ float quotient(float v, float scale, float y) {
    const float q = v * y;
    return fmaf(fmaf(-q, scale, v), y, q);
}
// Eight columns of a row to 8 bits; 16 lanes side by side have a block of columns.  All lanes of the warp; on: the columns are in the row's pitch.
__device__ __forceinline__ void quantise8(const RowsF8Args &a, size_t row, int c, bool on, const float (&n)[8]) {
    uint32_t most = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(n[e]) & 0x7FFFFFFFu);  // (what is undefined is larger than what is infinite)
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, off));
    const bool fine = most < 0x7F800000u;
    const float scale = fine ? __uint_as_float(most) / kMost : __uint_as_float(0x7FFFFFFFu);
    if (!on) return;
    if (c % kF8Block == 0) a.scales[static_cast<size_t>(c / kF8Block) * f8_scale_pitch(a.ntok) + row] = scale;
    uint2 q = make_uint2(0, 0);
    if (scale >= 0x1p-80f && scale <= 0x1p100f) {
        const float y = 1.0f / scale;
        q.x = pack2(quotient(n[0], scale, y), quotient(n[1], scale, y)) | pack2(quotient(n[2], scale, y), quotient(n[3], scale, y)) << 16;
        q.y = pack2(quotient(n[4], scale, y), quotient(n[5], scale, y)) | pack2(quotient(n[6], scale, y), quotient(n[7], scale, y)) << 16;
    } else if (fine && scale > 0.0f) {
        q.x = pack2(n[0] / scale, n[1] / scale) | pack2(n[2] / scale, n[3] / scale) << 16;
        q.y = pack2(n[4] / scale, n[5] / scale) | pack2(n[6] / scale, n[7] / scale) << 16;
    }
    *reinterpret_cast<uint2 *>(a.q + row * f8_pitch(a.cols) + c) = q;
}

// Without a norm the blocks of columns have nothing to do with one another: 16 lanes each, UNITS of them, wherever they lie.
template <typename T, int UNITS, bool VEC>
__global__ void __launch_bounds__(256) blocks_kernel(const RowsF8Args a, unsigned n_units, int row0) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ __align__(16) float s_turn[VEC ? 1 : 16 * kTurn];
    const unsigned n_blocks = static_cast<unsigned>(f8_blocks(a.cols)), step = gridDim.x * 16u, at = blockIdx.x * 16u + threadIdx.x / 16;
    float v[UNITS][8];
    unsigned row[UNITS];
    int c[UNITS];
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
        const unsigned unit = at + i * step;
        row[i] = unit / n_blocks;
        c[i] = unit < n_units ? static_cast<int>(unit - row[i] * n_blocks) * kF8Block + static_cast<int>(threadIdx.x & 15) * 8 : -1;
        row[i] += row0;
        values8<T, VEC>(a, row[i], c[i], s_turn, v[i]);
    }
#pragma unroll
    for (int i = 0; i < UNITS; ++i) quantise8(a, row[i], c[i], c[i] >= 0 && c[i] < f8_pitch(a.cols), v[i]);
}

__device__ __forceinline__ double over_block(double v, double *room) {  // (a warp, or all warps of the block)
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, off);
    if (blockDim.x > 32 && room != nullptr) {
        __syncthreads();
        if ((threadIdx.x & 31) == 0) room[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0.0;
        for (unsigned w = 0; w < blockDim.x / 32; ++w) v += room[w];
    }
    return v;
}

// With a norm: a row by a block, or (ONE_WARP) by each warp; values stay in registers, PARTS times eight of a thread.
template <typename T, int PARTS, bool ONE_WARP, bool VEC, int THREADS, int PER_SM>
__global__ void __launch_bounds__(THREADS, PER_SM) norm_kernel(const RowsF8Args a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ float s_sum[32];
    __shared__ double s_wide[32];
    __shared__ __align__(16) float s_turn[VEC ? 1 : THREADS / 16 * kTurn];
    const int lane = threadIdx.x & 31, threads = ONE_WARP ? 32 : static_cast<int>(blockDim.x), mine = ONE_WARP ? lane : static_cast<int>(threadIdx.x);
    const size_t row = ONE_WARP ? static_cast<size_t>(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32 : blockIdx.x;
    if (ONE_WARP && row >= static_cast<size_t>(a.ntok)) return;
    float v[PARTS][8];
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
        const int c = (i * threads + mine) * 8;
        values8<T, VEC>(a, row, c, s_turn, v[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(v[i][e], v[i][e], sum);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
    if constexpr (!ONE_WARP) {
        if (lane == 0) s_sum[threadIdx.x >> 5] = sum;
        __syncthreads();
        sum = 0.0f;
        for (int w = 0; w < threads / 32; ++w) sum += s_sum[w];
    }
    float factor = 0.0f;
    double wide_factor = 0.0;
    const bool wide = !(sum > 1e-30f && sum < 1e37f);  // squares that fp32 may not hold: in 64 bits
    if (wide) {
        double total = 0.0;
#pragma unroll
        for (int i = 0; i < PARTS; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) total = fma(static_cast<double>(v[i][e]), static_cast<double>(v[i][e]), total);
        wide_factor = 1.0 / sqrt(over_block(total, ONE_WARP ? nullptr : s_wide) / a.cols + static_cast<double>(a.eps));
    } else {
        factor = 1.0f / sqrtf(sum / static_cast<float>(a.cols) + a.eps);
    }
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
        const int c = (i * threads + mine) * 8;
        if (c < a.cols) {
            float g[8];
            load8(a.norm_w + c, a.cols - c, a.cols % 4 == 0, g);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = c + e >= a.cols ? 0.0f : wide ? static_cast<float>(static_cast<double>(v[i][e]) * wide_factor * static_cast<double>(g[e])) : v[i][e] * factor * g[e];
        }
        quantise8(a, row, c, c < f8_pitch(a.cols), v[i]);
    }
}

// Rows that registers do not hold: the values are made twice, their squares added up in 64 bits.
template <typename T, bool VEC>
__global__ void __launch_bounds__(1024) long_norm_kernel(const RowsF8Args a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ double s_wide[32];
    __shared__ __align__(16) float s_turn[VEC ? 1 : 64 * kTurn];
    const size_t row = blockIdx.x;
    double sum = 0.0;
    float v[8];
    for (int c0 = 0; c0 < a.cols; c0 += 8192) {
        values8<T, VEC>(a, row, c0 + static_cast<int>(threadIdx.x) * 8, s_turn, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fma(static_cast<double>(v[e]), static_cast<double>(v[e]), sum);
    }
    const double factor = 1.0 / sqrt(over_block(sum, s_wide) / a.cols + static_cast<double>(a.eps));
    RowsF8Args again = a;
    if (a.residual != nullptr) again.x = a.total, again.residual = nullptr;  // (what this thread has stored, as it reads them)
    for (int c0 = 0; c0 < a.cols; c0 += 8192) {
        const int c = c0 + static_cast<int>(threadIdx.x) * 8;
        values8<T, VEC>(again, row, c, s_turn, v);
        if (c < a.cols) {
            float g[8];
            load8(a.norm_w + c, a.cols - c, a.cols % 4 == 0, g);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = c + e >= a.cols ? 0.0f : static_cast<float>(static_cast<double>(v[e]) * factor * static_cast<double>(g[e]));
        }
        quantise8(a, row, c, c < f8_pitch(a.cols), v);
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

#ifndef NPARTS
#define NPARTS 1
#endif
template <typename T, bool VEC>
cudaError_t launch(const RowsF8Args &a, bool overlap, int sm_count, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[2];
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = launch_attributes(attr, overlap, 0);
    const int eights = static_cast<int>(f8_pitch(a.cols) / 8), n_blocks = f8_blocks(a.cols);
    if (a.norm_w == nullptr) {
        // (so many rows at a time that their blocks of columns can be counted in 32 bits)
        const int most = (1 << 30) / n_blocks;
        for (int row = 0; row < a.ntok; row += most) {
            const unsigned units = static_cast<unsigned>(most < a.ntok - row ? most : a.ntok - row) * static_cast<unsigned>(n_blocks), each = units >= 64u * static_cast<unsigned>(sm_count) ? 2 : 1;
            cfg.blockDim = dim3(256);
            cfg.gridDim = dim3((units + 16 * each - 1) / (16 * each));
            const cudaError_t err = each == 2 ? cudaLaunchKernelEx(&cfg, blocks_kernel<T, 2, VEC>, a, units, row) : cudaLaunchKernelEx(&cfg, blocks_kernel<T, 1, VEC>, a, units, row);
            if (err != cudaSuccess) return err;
        }
        return cudaSuccess;
    }
    if (eights <= 32) {
        cfg.blockDim = dim3(128);
        cfg.gridDim = dim3(static_cast<unsigned>((a.ntok + 3ll) / 4));
        return cudaLaunchKernelEx(&cfg, norm_kernel<T, 1, true, VEC, 128, 8>, a);
    }
    cfg.gridDim = dim3(static_cast<unsigned>(a.ntok));
    auto threads = [&](int parts) { return static_cast<unsigned>(((eights + parts - 1) / parts + 31) / 32 * 32); };
    int parts = a.ntok > 2 * sm_count ? NPARTS : 1;
    while (parts < 4 && threads(parts) > 1024) parts *= 2;
    cfg.blockDim = dim3(threads(parts));
    if (parts == 1) return threads(1) <= 640 ? cudaLaunchKernelEx(&cfg, norm_kernel<T, 1, false, VEC, 640, 2>, a) : cudaLaunchKernelEx(&cfg, norm_kernel<T, 1, false, VEC, 1024, 2>, a);
    if (parts == 2) return threads(2) <= 640 ? cudaLaunchKernelEx(&cfg, norm_kernel<T, 2, false, VEC, 640, 2>, a) : cudaLaunchKernelEx(&cfg, norm_kernel<T, 2, false, VEC, 1024, 1>, a);
    if (threads(4) <= 576) return cudaLaunchKernelEx(&cfg, norm_kernel<T, 4, false, VEC, 576, 2>, a);
    if (threads(4) <= 1024) return cudaLaunchKernelEx(&cfg, norm_kernel<T, 4, false, VEC, 1024, 1>, a);
    cfg.blockDim = dim3(1024);
    return cudaLaunchKernelEx(&cfg, long_norm_kernel<T, VEC>, a);
}
template <typename T>
cudaError_t launch(const RowsF8Args &a, bool overlap, int sm_count, cudaStream_t stream) {
    return a.cols % (16 / static_cast<int>(sizeof(T))) == 0 ? launch<T, true>(a, overlap, sm_count, stream) : launch<T, false>(a, overlap, sm_count, stream);
}

}  // namespace

cudaError_t launch_rows_f8(const RowsF8Args &a, bool overlap, int sm_count, cudaStream_t stream) {
    return a.elem == 2 ? launch<__half>(a, overlap, sm_count, stream) : launch<float>(a, overlap, sm_count, stream);
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
