// Activation rows in 8-bit floating point (e4m3) with a scale for each 128 columns, after what a layer does to them on the way to a projection:
//   v = x,  or silu(x) * x2,  or h = x + residual (rounded to its type and stored);   n = v * g / sqrt(mean(v^2) + eps), or v;
//   s = max |n| / 448 over 128 columns, in fp32,   q = n / s (in fp32) rounded to the nearest e4m3 value, ties to even.
//
// Each value is read once and stays in registers: 16 of a thread, 8 threads for a block of columns, whose largest three shuffles find.  Norms take a block per row (a warp, up to
// 512 columns), everything else takes blocks of columns wherever they lie.
// What bounds it: fp32 rows the memory, fp16 ones the instructions (issue slots 60 to 74 %).  4001 x 5120, fp32 and fp16: residual and norm 41 us (6.5 TB/s) and 32 (4.5), gated 29
// (6.5) and 26 (3.9), neither 18 (5.8) and 13 (4.8).  With 8 values of a thread and a division each: 56 and 58, 42 and 46, 23 and 24.  1 x 5120 3 to 4.5, 77 x 17408
// gated 3.3.
#include <cuda_fp16.h>

#include "vqm_kernels.h"
#include "vqm_packed.cuh"

namespace vqm {
namespace {

constexpr float kMost = 448.0f;  // of e4m3

// silu(x) * x2.  With h = exp(-|x| / 2) neither a far negative x, whose silu is exp(x) x, nor a large x2 leaves fp32 on the way.  h = 2^t (1 + d), where t is the
// argument in fp32 and d what its rounding has left, times ln 2.  (x below -174 counts as gated off; what is undefined comes back with x itself.)
__device__ __forceinline__ float gated(float x, float x2) {
    constexpr float kHalfLog2e = 0.72134752044448170f, kRest = static_cast<float>(0.72134752044448170368 - static_cast<double>(kHalfLog2e)), kLn2 = 0.69314718055994531f;
    const float y = fmaxf(-fabsf(x), -400.0f), t = y * kHalfLog2e, d = fmaf(y, kRest, fmaf(y, kHalfLog2e, -t));
    float h, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(h) : "f"(t));
    h = fmaf(h, d * kLn2, h);
    const float g = x < 0.0f ? h : 1.0f;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(h, h, 1.0f)));
    return x * g * r * (x2 * g);
}

// Two values as e4m3, the first in the lower byte; what is beyond 448 becomes that.
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    uint16_t out;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(out) : "f"(b), "f"(a));
    return out;
}

constexpr int kEach = 16;                 // values of a thread
constexpr int kLanes = kF8Block / kEach;  // threads of a block of columns
// They are groups of as many as 16 bytes hold; a group of each of the kLanes threads, then the next group of each: what is read or written together lies together.
template <typename T>
constexpr int kGroup = 16 / static_cast<int>(sizeof(T));
template <typename T>
__device__ __forceinline__ int column(int e) {  // of a thread's value e, in its block of columns
    constexpr int G = kGroup<T>;
    return e / G * G * kLanes + static_cast<int>(threadIdx.x % kLanes) * G + e % G;
}

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float rounded(float v, const float *) { return v; }
__device__ __forceinline__ __half rounded(float v, const __half *) { return __float2half_rn(v); }
__device__ __forceinline__ void load(const float *p, float *v) {
    const float4 x = *reinterpret_cast<const float4 *>(p);
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
}
__device__ __forceinline__ void load(const __half *p, float *v) {
    const uint4 w = *reinterpret_cast<const uint4 *>(p);
    const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&r[e]));
        v[2 * e] = f.x, v[2 * e + 1] = f.y;
    }
}
// Rounds the values to the buffer's type, and stores them.
__device__ __forceinline__ void store(float *p, float *v) { *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void store(__half *p, float *v) {
    uint32_t r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const __half2 h = __floats2half2_rn(v[2 * e], v[2 * e + 1]);
        r[e] = *reinterpret_cast<const uint32_t *>(&h);
        const float2 f = __half22float2(h);
        v[2 * e] = f.x, v[2 * e + 1] = f.y;
    }
    *reinterpret_cast<uint4 *>(p) = make_uint4(r[0], r[1], r[2], r[3]);
}

// A thread's values of the block of columns from c0 on, before the norm, zeros behind the row's last; the sums are stored.  By all lanes of a warp; c0 < 0: none.
// VEC: rows begin on 16 bytes, so groups are whole.  Others are read (and sums written) kLanes columns after kLanes columns, and turned in shared memory.
constexpr int kTurn = kF8Block + kLanes;  // floats of a block of columns (the others' in other banks)
template <typename T, bool VEC>
__device__ __forceinline__ void values(const RowsF8Args &a, size_t row, int c0, float *room, float (&v)[kEach]) {
    const size_t at = row * a.cols;
    const T *x = static_cast<const T *>(a.x) + at, *second = static_cast<const T *>(a.residual != nullptr ? a.residual : a.x2) + at;
    T *total = static_cast<T *>(a.total) + at;
    if constexpr (VEC) {
        constexpr int G = kGroup<T>;
        float more[kEach];
        int c[kEach / G];
#pragma unroll
        for (int g = 0; g < kEach / G; ++g) {
            c[g] = c0 >= 0 && c0 + column<T>(g * G) < a.cols ? c0 + column<T>(g * G) : -1;
#pragma unroll
            for (int e = 0; e < G; ++e) v[g * G + e] = more[g * G + e] = 0.0f;
            if (c[g] >= 0) load(x + c[g], v + g * G);
        }
        if (a.residual != nullptr || a.x2 != nullptr)
#pragma unroll
            for (int g = 0; g < kEach / G; ++g)
                if (c[g] >= 0) load(second + c[g], more + g * G);
        if (a.residual != nullptr) {
#pragma unroll
            for (int e = 0; e < kEach; ++e) v[e] += more[e];
#pragma unroll
            for (int g = 0; g < kEach / G; ++g)
                if (c[g] >= 0) store(total + c[g], v + g * G);
        } else if (a.x2 != nullptr) {
#pragma unroll
            for (int e = 0; e < kEach; ++e) v[e] = gated(v[e], more[e]);
        }
    } else {
        const int lane = static_cast<int>(threadIdx.x % kLanes), c = (c0 < 0 ? a.cols : c0) + lane;
        float *const turn = room + threadIdx.x / kLanes * kTurn;
        float more[kEach] = {};
#pragma unroll
        for (int e = 0; e < kEach; ++e) v[e] = c + e * kLanes < a.cols ? as_float(x[c + e * kLanes]) : 0.0f;
        if (a.residual != nullptr || a.x2 != nullptr)
#pragma unroll
            for (int e = 0; e < kEach; ++e) more[e] = c + e * kLanes < a.cols ? as_float(second[c + e * kLanes]) : 0.0f;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            if (a.residual != nullptr) {
                const T sum = rounded(v[e] + more[e], static_cast<const T *>(nullptr));
                if (c + e * kLanes < a.cols) total[c + e * kLanes] = sum;
                v[e] = as_float(sum);
            } else if (a.x2 != nullptr) {
                v[e] = gated(v[e], more[e]);
            }
            turn[lane + e * kLanes] = v[e];
        }
        __syncwarp();
#pragma unroll
        for (int e = 0; e < kEach; e += 4) {
            const float4 p = *reinterpret_cast<const float4 *>(turn + column<T>(e));
            v[e] = p.x, v[e + 1] = p.y, v[e + 2] = p.z, v[e + 3] = p.w;
        }
        __syncwarp();
    }
}
// The norm's weights of a thread's values, zeros behind the last.
template <typename T, bool VEC>
__device__ __forceinline__ void weights(const RowsF8Args &a, int c0, float (&g)[kEach]) {
#pragma unroll
    for (int e = 0; e < kEach; e += 4) {
        const int c = c0 + column<T>(e);
        if (VEC ? c < a.cols : c + 4 <= a.cols) {  // (buffers and tensors are 16-byte aligned)
            load(a.norm_w + c, g + e);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) g[e + i] = !VEC && c + i < a.cols ? a.norm_w[c + i] : 0.0f;
        }
    }
}
// v / scale as fp32 rounds it.  With y = 1 / scale rounded, q = v y and the remainder v - q scale (which one fused multiply and add gives exactly), q + remainder y rounds
// to that (P. Markstein, IBM J. Res. Dev. 34, 1990) wherever nothing of it underflows: for q of 2^-10 on, and smaller ones are nothing in e4m3, where scale is in [2^-80, 2^100].
__device__ __forceinline__ float quotient(float v, float scale, float y) {
    const float q = v * y;
    return fmaf(fmaf(-q, scale, v), y, q);
}
__device__ __forceinline__ Two quotients(Two v, Two minus_scale, Two y) {
    const Two q = mul2(v, y);
    return fma2(fma2(q, minus_scale, v), y, q);
}
// The largest magnitude; what is undefined stays so.
__device__ __forceinline__ float most_of(float a, float b) {
    float v;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(fabsf(a)), "f"(fabsf(b)));
    return v;
}
// A thread's values of the block of columns from c0 on to 8 bits.  All lanes of the warp; c0 < 0, or beyond the row's last: none.
template <typename T>
__device__ __forceinline__ void quantise(const RowsF8Args &a, size_t row, int c0, const float (&n)[kEach]) {
    float m[kEach / 2];
#pragma unroll
    for (int e = 0; e < kEach / 2; ++e) m[e] = most_of(n[e], n[e + kEach / 2]);
#pragma unroll
    for (int w = kEach / 4; w > 0; w /= 2)
#pragma unroll
        for (int e = 0; e < w; ++e) m[e] = most_of(m[e], m[e + w]);
    float most = m[0];
#pragma unroll
    for (int off = kLanes / 2; off > 0; off >>= 1) most = most_of(most, __shfl_xor_sync(0xFFFFFFFFu, most, off));
    if (c0 < 0 || c0 >= a.cols) return;
    float scale = quotient(most, kMost, 1.0f / kMost);
    uint32_t q[kEach / 4] = {};
    if (scale >= 0x1p-80f && scale <= 0x1p100f) {
        const float y = 1.0f / scale;
        const Two yy = two(y, y), minus = two(-scale, -scale);
#pragma unroll
        for (int i = 0; i < kEach / 4; ++i) {
            float t[4];
            both(quotients(two(n[4 * i], n[4 * i + 1]), minus, yy), t[0], t[1]);
            both(quotients(two(n[4 * i + 2], n[4 * i + 3]), minus, yy), t[2], t[3]);
            q[i] = pack2(t[0], t[1]) | pack2(t[2], t[3]) << 16;
        }
    } else {
        scale = most < INFINITY ? most / kMost : __uint_as_float(0x7FFFFFFFu);
        if (scale > 0.0f)
#pragma unroll
            for (int i = 0; i < kEach / 4; ++i)
                q[i] = pack2(n[4 * i] / scale, n[4 * i + 1] / scale) | pack2(n[4 * i + 2] / scale, n[4 * i + 3] / scale) << 16;
    }
    if (threadIdx.x % kLanes == 0) a.scales[static_cast<size_t>(c0 / kF8Block) * f8_scale_pitch(a.ntok) + row] = scale;
    uint8_t *const to = a.q + row * f8_pitch(a.cols) + c0;
    const int left = static_cast<int>(f8_pitch(a.cols)) - c0;  // (a multiple of 16)
    if constexpr (kGroup<T> == 8) {
#pragma unroll
        for (int g = 0; g < 2; ++g)
            if (column<T>(8 * g) < left) *reinterpret_cast<uint2 *>(to + column<T>(8 * g)) = make_uint2(q[2 * g], q[2 * g + 1]);
    } else {
#pragma unroll
        for (int g = 0; g < 4; ++g)
            if (column<T>(4 * g) < left) *reinterpret_cast<uint32_t *>(to + column<T>(4 * g)) = q[g];
    }
}

constexpr int kBlocksThreads = 256;
// Without a norm the blocks of columns have nothing to do with one another: kLanes threads each, wherever they lie.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kBlocksThreads, 5) blocks_kernel(const RowsF8Args a, unsigned n_units, int row0) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ __align__(16) float s_turn[VEC ? 1 : kBlocksThreads / kLanes * kTurn];
    const unsigned n_blocks = static_cast<unsigned>(f8_blocks(a.cols)), unit = blockIdx.x * (kBlocksThreads / kLanes) + threadIdx.x / kLanes, row = unit / n_blocks;
    const int c0 = unit < n_units ? static_cast<int>(unit - row * n_blocks) * kF8Block : -1;
    float v[kEach];
    values<T, VEC>(a, row0 + row, c0, s_turn, v);
    quantise<T>(a, row0 + row, c0, v);
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

// With a norm: a row by a block, or (ONE_WARP) by each warp; values stay in registers, PARTS times kEach of a thread.
template <typename T, int PARTS, bool ONE_WARP, bool VEC, int THREADS, int PER_SM>
__global__ void __launch_bounds__(THREADS, PER_SM) norm_kernel(const RowsF8Args a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ float s_sum[32];
    __shared__ double s_wide[32];
    __shared__ __align__(16) float s_turn[VEC ? 1 : THREADS / kLanes * kTurn];
    const int lane = threadIdx.x & 31, threads = ONE_WARP ? 32 : static_cast<int>(blockDim.x), mine = ONE_WARP ? lane : static_cast<int>(threadIdx.x);
    const size_t row = ONE_WARP ? static_cast<size_t>(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32 : blockIdx.x;
    if (ONE_WARP && row >= static_cast<size_t>(a.ntok)) return;
    float v[PARTS][kEach];
    Two squares = 0;
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
        values<T, VEC>(a, row, (i * threads + mine) / kLanes * kF8Block, s_turn, v[i]);
#pragma unroll
        for (int e = 0; e < kEach; e += 2) {
            const Two x = two(v[i][e], v[i][e + 1]);
            squares = fma2(x, x, squares);
        }
    }
    float sum, other;
    both(squares, sum, other);
    sum += other;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
    if constexpr (!ONE_WARP) {
        if (lane == 0) s_sum[threadIdx.x >> 5] = sum;
        __syncthreads();
        sum = 0.0f;
        for (int w = 0; w < threads / 32; ++w) sum += s_sum[w];
    }
    if (sum > 1e-30f && sum < 1e37f) {
        const float factor = 1.0f / sqrtf(sum / static_cast<float>(a.cols) + a.eps);
        const Two f = two(factor, factor);
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            const int c0 = (i * threads + mine) / kLanes * kF8Block;
            if (c0 < a.cols) {
                float g[kEach];
                weights<T, VEC>(a, c0, g);
#pragma unroll
                for (int e = 0; e < kEach; e += 2) both(mul2(mul2(two(v[i][e], v[i][e + 1]), f), two(g[e], g[e + 1])), v[i][e], v[i][e + 1]);
            }
            quantise<T>(a, row, c0, v[i]);
        }
    } else {  // squares that fp32 may not hold: in 64 bits
        double total = 0.0;
#pragma unroll
        for (int i = 0; i < PARTS; ++i)
#pragma unroll
            for (int e = 0; e < kEach; ++e) total = fma(static_cast<double>(v[i][e]), static_cast<double>(v[i][e]), total);
        const double factor = 1.0 / sqrt(over_block(total, ONE_WARP ? nullptr : s_wide) / a.cols + static_cast<double>(a.eps));
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            const int c0 = (i * threads + mine) / kLanes * kF8Block;
            if (c0 < a.cols) {
                float g[kEach];
                weights<T, VEC>(a, c0, g);
#pragma unroll
                for (int e = 0; e < kEach; ++e) v[i][e] = c0 + column<T>(e) < a.cols ? static_cast<float>(static_cast<double>(v[i][e]) * factor * static_cast<double>(g[e])) : 0.0f;
            }
            quantise<T>(a, row, c0, v[i]);
        }
    }
}

// Rows that registers do not hold: the values are made twice, their squares added up in 64 bits.
template <typename T, bool VEC>
__global__ void __launch_bounds__(1024) long_norm_kernel(const RowsF8Args a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ double s_wide[32];
    extern __shared__ __align__(16) float s_long_turn[];
    const size_t row = blockIdx.x;
    const int step = static_cast<int>(blockDim.x) * kEach, first = static_cast<int>(threadIdx.x) / kLanes * kF8Block;
    double sum = 0.0;
    float v[kEach];
    for (int c = 0; c < a.cols; c += step) {
        values<T, VEC>(a, row, c + first, s_long_turn, v);
#pragma unroll
        for (int e = 0; e < kEach; ++e) sum = fma(static_cast<double>(v[e]), static_cast<double>(v[e]), sum);
    }
    const double factor = 1.0 / sqrt(over_block(sum, s_wide) / a.cols + static_cast<double>(a.eps));
    RowsF8Args again = a;
    if (a.residual != nullptr) again.x = a.total, again.residual = nullptr;  // (what this thread has stored, as it reads them)
    for (int c = 0; c < a.cols; c += step) {
        const int c0 = c + first;
        values<T, VEC>(again, row, c0, s_long_turn, v);
        if (c0 < a.cols) {
            float g[kEach];
            weights<T, VEC>(a, c0, g);
#pragma unroll
            for (int e = 0; e < kEach; ++e) v[e] = c0 + column<T>(e) < a.cols ? static_cast<float>(static_cast<double>(v[e]) * factor * static_cast<double>(g[e])) : 0.0f;
        }
        quantise<T>(a, row, c0, v);
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

template <typename T, bool VEC>
cudaError_t launch(const RowsF8Args &a, bool overlap, int sm_count, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[2];
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = launch_attributes(attr, overlap, 0);
    const int n_blocks = f8_blocks(a.cols), pieces = n_blocks * kLanes;
    if (a.norm_w == nullptr) {
        // (so many rows at a time that their blocks of columns can be counted in 32 bits)
        const int most = (1 << 30) / n_blocks;
        for (int row = 0; row < a.ntok; row += most) {
            const unsigned units = static_cast<unsigned>(most < a.ntok - row ? most : a.ntok - row) * static_cast<unsigned>(n_blocks);
            constexpr unsigned kAtOnce = kBlocksThreads / kLanes;
            cfg.blockDim = dim3(kBlocksThreads);
            cfg.gridDim = dim3((units + kAtOnce - 1) / kAtOnce);
            const cudaError_t err = cudaLaunchKernelEx(&cfg, blocks_kernel<T, VEC>, a, units, row);
            if (err != cudaSuccess) return err;
        }
        return cudaSuccess;
    }
    if (pieces <= 32) {
        cfg.blockDim = dim3(128);
        cfg.gridDim = dim3(static_cast<unsigned>((a.ntok + 3ll) / 4));
        return cudaLaunchKernelEx(&cfg, norm_kernel<T, 1, true, VEC, 128, 8>, a);
    }
    cfg.gridDim = dim3(static_cast<unsigned>(a.ntok));
    auto threads = [&](int parts) { return static_cast<unsigned>(((pieces + parts - 1) / parts + 31) / 32 * 32); };
    auto norm = [&](auto kernel, int parts) {
        cfg.blockDim = dim3(threads(parts));
        return cudaLaunchKernelEx(&cfg, kernel, a);
    };
    // Blocks per SM: as many as leave the values in registers, 16-bit ones, which wait for less, one more (4001 x 5120 with residual: fp32 41 us with three, 43 with four and 44 with
    // two; fp16 35, 32 and 45).  Few rows do not fill the SMs anyhow.
    constexpr int kPerSm = VEC && sizeof(T) == 2 ? 4 : 3;
    const bool few = a.ntok <= 2 * sm_count;
    if (threads(1) <= 384 && !few) return norm(norm_kernel<T, 1, false, VEC, 384, kPerSm>, 1);
    if (threads(1) <= 512 && few) return norm(norm_kernel<T, 1, false, VEC, 512, 1>, 1);
    if (threads(2) <= 512) return norm(norm_kernel<T, 2, false, VEC, 512, 2>, 2);
    if (threads(3) <= 384) return norm(norm_kernel<T, 3, false, VEC, 384, 2>, 3);
    if (threads(4) <= 512) return norm(norm_kernel<T, 4, false, VEC, 512, 1>, 4);
    cfg.blockDim = dim3(512);
    cfg.dynamicSmemBytes = VEC ? 0 : 512 / kLanes * kTurn * sizeof(float);
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
