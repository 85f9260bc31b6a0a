// Activation rows as 8-bit integers with a scale per row, after what a layer does to them on the way to a projection:
//   v = x,  or silu(x) * x2,  or h = x + residual (rounded to its type and stored);   n = v * g / sqrt(mean(v^2) + eps), or v;
//   s = max |n| / 127 in fp32,   q = n / s rounded to the nearest whole number, ties to even.
// Which of two whole numbers a value goes to is decided by the formula, not by the order of 32-bit roundings: the mean and the largest value are
// taken in 64 bits (the mean's square root cancels out of n / s but for the rounding of s), the values in 32, and a value that 32 bits leave next to a
// half is worked out again in 64.
//
// A block per row (of 32 to 1024 threads), its values in registers (but for some that long rows spill, see blocks_per_sm): memory is read and written once.
// Rows too long for that (more than 24564 values), norms of gated values, and rows whose largest value is out of fp32's middle range are worked out in 64
// bits throughout, norms of up to 20480 gated values with each value made once.
//
// What bounds it: 4001 rows of 5120 with residual and norm take 52 us in fp32 (5080 GB/s of the 6550 that a copy gets) and 34 to 37 in fp16 (3900 GB/s).  There,
// and in gated rows (4001 x 5120 38 us in both types, 1000 x 17408 49 in fp32 and 37 in fp16), neither the issue slots (32 to 52 %) nor DRAM (23 to 35 %) are
// at their limit: a row's steps follow one another, with two barriers and one thread's 64-bit work between its two passes over the registers, and the rows
// that an SM holds cover a part of that.  Lengths that are no multiple of 4 write bytes one by one (4001 x 5121 58 to 77 us).  One row: 3.4 us.  In 64 bits:
// 1000 gated rows of 28672 458 us in fp32, without a gate 382 with norm and 224 plain; norms of gated rows 371 (4001 x 5120) and 296 (1000 x 17408).
// What it took: more rows at a time on an SM (below); an error bound of the gate that looks at the values, so that fewer of them are worked out in 64 bits (1000
// gated rows of 17408 57 and 52 us, 4001 of 5120 in fp16 53 and 38).
// Tried: rows copied ahead into shared memory by blocks that stay (71 us for 47), four values looked at together for nearness to a half (no gain).
#include <cuda_fp16.h>

#include "vqm_kernels.h"

namespace vqm {
namespace {

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ void put(float *p, float v) { *p = v; }
__device__ __forceinline__ void put(__half *p, float v) { *p = __float2half_rn(v); }

__device__ __forceinline__ void load4(const float *p, float (&v)[4]) {
    const float4 w = *reinterpret_cast<const float4 *>(p);
    v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
}

constexpr int kMostFast = 24564;  // columns of a row that 512 threads hold in 12 vectors each, or 1024 in 6, wherever it begins; longer ones take 5 to 10 times as long per value
constexpr float kUndefined = __builtin_nanf("");
constexpr double kMostScale = 3.4028235677973366e38;  // half a step above fp32's largest: rounds to infinity from here on

struct RowShared {
    double d[32];
    float a[32];
    int bad;
    unsigned long long largest;  // bits of a positive number, which are in its order
    double r, scale;
    float factor;
};

// One row by the whole block, in 64 bits.
template <typename T>
static __device__ __noinline__ void exact_row(const RowsI8Args &a, size_t row, bool total_is_there, RowShared &s) {
    const size_t at = row * a.cols;
    const T *x = static_cast<const T *>(a.x) + at, *x2 = static_cast<const T *>(a.x2) + at, *res = static_cast<const T *>(a.residual) + at;
    T *total = static_cast<T *>(a.total) + at;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, threads = static_cast<int>(blockDim.x);
    auto value = [&](int c) -> double {
        if (a.residual != nullptr) return as_float(total[c]);  // (by the thread that wrote it)
        const double v = as_float(x[c]);
        return a.x2 != nullptr ? v / (1.0 + exp(-v)) * static_cast<double>(as_float(x2[c])) : v;
    };
    auto combine = [&](double v, auto op) -> double {
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, off));
        __syncthreads();
        if (lane == 0) s.d[warp] = v;
        __syncthreads();
        v = s.d[0];
        for (int i = 1; i < threads / 32; ++i) v = op(v, s.d[i]);
        return v;
    };
    if (total_is_there) __syncthreads();  // (the threads of the fast pass hold other columns)
    else if (a.residual != nullptr)
        for (int c = threadIdx.x; c < a.cols; c += threads) put(total + c, as_float(x[c]) + as_float(res[c]));
    double r = 1.0;
    if (a.norm_w != nullptr) {
        double sum = 0.0;
        for (int c = threadIdx.x; c < a.cols; c += threads) {
            const double v = value(c);
            sum += v * v;
        }
        sum = combine(sum, [](double p, double q) { return p + q; });
        r = 1.0 / sqrt(sum / a.cols + static_cast<double>(a.eps));
    }
    if (threadIdx.x == 0) s.bad = 0;
    double top = 0.0;
    bool bad = false;
    for (int c = threadIdx.x; c < a.cols; c += threads) {
        const double n = a.norm_w != nullptr ? value(c) * r * static_cast<double>(a.norm_w[c]) : value(c);
        bad |= !(fabs(n) <= 1e300);
        top = fmax(top, fabs(n));
    }
    top = combine(top, [](double p, double q) { return fmax(p, q); });
    if (bad) s.bad = 1;
    __syncthreads();
    // a value that is infinite or undefined makes the row's outputs undefined
    const float scale = s.bad || top / 127.0 >= kMostScale ? kUndefined : static_cast<float>(top / 127.0);
    if (threadIdx.x == 0) a.scales[row] = scale;
    const long long pitch = i8_pitch(a.cols);
    for (int c = threadIdx.x; c < pitch; c += threads) {
        int q = 0;
        if (c < a.cols && scale > 0.0f) {
            const double n = a.norm_w != nullptr ? value(c) * r * static_cast<double>(a.norm_w[c]) : value(c);
            q = min(127, max(-127, __double2int_rn(n / static_cast<double>(scale))));
        }
        a.q[row * pitch + c] = static_cast<int8_t>(q);
    }
}

template <typename T>
__global__ void __launch_bounds__(512) exact_rows_kernel(const RowsI8Args a) {
    __shared__ RowShared s;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    exact_row<T>(a, blockIdx.x, false, s);
}

// The norm of gated values, whose mean wants more digits than 32 bits leave of silu: in 64 bits too, but each value is made once and kept.
template <typename T, int NV>
__global__ void __launch_bounds__(512) gated_norm_kernel(const RowsI8Args a) {
    __shared__ double s_sum[16], s_top[16];
    const size_t row = blockIdx.x, at = row * a.cols;
    const T *x = static_cast<const T *>(a.x) + at, *x2 = static_cast<const T *>(a.x2) + at;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    double v[NV], sum = 0.0, top = 0.0;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = static_cast<int>(threadIdx.x) + i * 512;
        v[i] = 0.0;
        if (c < a.cols) {
            const double e = static_cast<double>(as_float(x[c]));
            v[i] = e / (1.0 + exp(-e)) * static_cast<double>(as_float(x2[c]));
        }
        sum = fma(v[i], v[i], sum);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = static_cast<int>(threadIdx.x) + i * 512;
        if (c < a.cols) v[i] *= static_cast<double>(a.norm_w[c]);
        bad |= !(fabs(v[i]) <= 1e300);
        top = fmax(top, fabs(v[i]));
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off), top = fmax(top, __shfl_xor_sync(0xffffffffu, top, off));
    if (__any_sync(0xffffffffu, bad)) top = __longlong_as_double(0x7ff0000000000000ll);
    if (lane == 0) s_sum[warp] = sum, s_top[warp] = top;
    __syncthreads();
    sum = lane < 16 ? s_sum[lane] : 0.0, top = lane < 16 ? s_top[lane] : 0.0;
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off), top = fmax(top, __shfl_xor_sync(0xffffffffu, top, off));
    sum = __shfl_sync(0xffffffffu, sum, 0), top = __shfl_sync(0xffffffffu, top, 0);
    const double r = 1.0 / sqrt(sum / a.cols + static_cast<double>(a.eps)), wide = top * r / 127.0;
    const float scale = wide < kMostScale ? static_cast<float>(wide) : kUndefined;  // (not so for undefined ones)
    if (threadIdx.x == 0) a.scales[row] = scale;
    const double factor = r / static_cast<double>(scale);
    const long long pitch = i8_pitch(a.cols);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = static_cast<int>(threadIdx.x) + i * 512;
        if (c >= pitch) continue;
        const int q = scale > 0.0f && c < a.cols ? min(127, max(-127, __double2int_rn(v[i] * factor))) : 0;
        a.q[row * pitch + c] = static_cast<int8_t>(q);
    }
}

// silu(x) * y in 64 bits
static __device__ __noinline__ double exact_gate(float x, float y) { return static_cast<double>(x) / (1.0 + exp(-static_cast<double>(x))) * static_cast<double>(y); }

// n / s as a whole number, n = d r, in 64 bits (divided: a tie stays a tie)
static __device__ __noinline__ int exact_whole(double d, double r, double scale) { return __double2int_rn(d * r / scale); }

// 1 / (1 + exp(-x)), off by no more than 5e-7 + 7.5e-8 max(-x, 0): 2^-22 of ex2, 2^-24 |x| of its argument and 1.4e-8 |x| of the constant in it, 2^-24 of the
// sum, 2^-23 of the reciprocal.
__device__ __forceinline__ float sigmoid(float x) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * -1.44269504f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return r;
}

__device__ __forceinline__ float largest_of(float a, float b) {  // undefined if either is
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}

// r such that r r m = 1, in 64 bits: two steps of Newton's method from 22 bits
__device__ __forceinline__ double inverse_root(double m) {
    if (!(m > 1e-30 && m < 1e30)) return 1.0 / sqrt(m);
    double r = static_cast<double>(rsqrtf(static_cast<float>(m)));
    const double half = 0.5 * m;
    r = fma(r, fma(-half * r, r, 0.5), r);
    return fma(r, fma(-half * r, r, 0.5), r);
}

// Four values in registers: as they come, or as floats where they are no longer of the buffer's type.
template <typename T, bool WIDE>
struct Kept {
    float f[4];
    __device__ __forceinline__ void fetch(const T *p);
    __device__ __forceinline__ void values(float (&v)[4]) const {
#pragma unroll
        for (int l = 0; l < 4; ++l) v[l] = f[l];
    }
    __device__ __forceinline__ void keep(const float (&v)[4]) {
#pragma unroll
        for (int l = 0; l < 4; ++l) f[l] = v[l];
    }
    __device__ __forceinline__ void put_to(float *p) const { *reinterpret_cast<float4 *>(p) = make_float4(f[0], f[1], f[2], f[3]); }
    __device__ __forceinline__ void add(const Kept &y) {
#pragma unroll
        for (int l = 0; l < 4; ++l) f[l] += y.f[l];
    }
};
template <>
struct Kept<__half, false> {
    uint2 w;
    __device__ __forceinline__ void fetch(const __half *p) { w = *reinterpret_cast<const uint2 *>(p); }
    __device__ __forceinline__ void values(float (&v)[4]) const {
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&w.y));
        v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
    }
    __device__ __forceinline__ void keep(const float (&v)[4]) {
        const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
        w = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    }
    __device__ __forceinline__ void put_to(__half *p) const { *reinterpret_cast<uint2 *>(p) = w; }
    // (one rounding, as of the fp32 sum: its 24 bits are twice 11 and two more)
    __device__ __forceinline__ void add(const Kept &y) {
        const __half2 a = __hadd2_rn(*reinterpret_cast<const __half2 *>(&w.x), *reinterpret_cast<const __half2 *>(&y.w.x));
        const __half2 b = __hadd2_rn(*reinterpret_cast<const __half2 *>(&w.y), *reinterpret_cast<const __half2 *>(&y.w.y));
        w = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    }
};
template <typename T, bool WIDE>
__device__ __forceinline__ void Kept<T, WIDE>::fetch(const T *p) {
    if constexpr (sizeof(T) == 4) {
        load4(reinterpret_cast<const float *>(p), f);
    } else {
        Kept<__half, false> half;
        half.fetch(reinterpret_cast<const __half *>(p));
        half.values(f);
    }
}

// Blocks that an SM holds at least, which bounds the registers: while some rows wait for memory, others are worked on.  A bound that makes threads spill some
// registers still pays where the blocks it gains are a large part, and does not where 100 bytes and more are spilled for a third one of long fp32 rows.
// Measured, us, against one block less or more; in brackets bytes spilled by plain and gated variants of rows that are multiples of 4 (others spill more):
//   fp16, 128 threads           7 [48 and 116 at most]: norm 4001 x 5120 36.7 (6: 38.0), gated 38.2 (6: 40.2), 4001 x 4096 gated 34.4 (6: 33.0)
//   fp16, 256 threads           4 up to 10 vectors [92, 120]: gated 2000 x 8192 30.1 (3: 34.2), 1000 x 10000 23.2 (3: 24.4), norm 26.8 (3: 26.0)
//                               3 for 12 vectors [0, 84]: gated 1000 x 12000 30.6 (4: 35.3), 400 x 12000 12.8 (4: 19.0); but rows of odd lengths 4: 12001 43.0 (3: 48.4)
//   fp16, 512 threads           2 [120, 160]: gated 1000 x 17408 36.7 (1: 50.9), norm 39.3 (1: 47.4), 1000 x 14336 31.2 (1: 45.3)
//   fp32, 256 threads           4 for 5 vectors [12, 0]: norm 4001 x 5120 52.7 (3 took 2 us more); 3 for 8 [24, 0] (4 spills more)
//                               2 for 10 and 12 [0, 0]: 1000 x 10000 gated 28.9, norm 36, plain 16.2 (3: 33.3, 42.5, 15.1), 1000 x 12000 33.5, 44, 18.2 (3: 46.1, 59, 17.6);
//                               400 x 10000, which 3 hold at once, gated 15.8 (3: 13.6)
template <typename T, int NV, int THREADS, bool LOOSE>
constexpr int blocks_per_sm() {
    if (THREADS == 512) return 2;
    if (THREADS == 256 && sizeof(T) == 2) return NV <= 10 || LOOSE ? 4 : 3;
    if (THREADS == 256) return NV <= 5 ? 4 : NV <= 8 ? 3 : 2;
    return THREADS == 128 && sizeof(T) == 2 ? 7 : 1;
}

// A block per row.  A thread holds NV vectors of 4 neighbouring columns, vector i at (thread + i * threads) * 4: v before the norm's weights, which come
// from the caches both times.  LOOSE: rows of any length, whose vectors lie on the buffers' grid, not the row's: the first and the last may be
// partly outside of the row, and the norm's weights and the outputs, which lie on other grids, go one by one.
template <typename T, int NV, int THREADS, bool GATED, bool LOOSE>
__global__ void __launch_bounds__(THREADS, blocks_per_sm<T, NV, THREADS, LOOSE>()) rows_i8_kernel(const RowsI8Args a) {
    __shared__ RowShared s;
    constexpr int WARPS = THREADS / 32;
    const size_t row = blockIdx.x, at = row * a.cols;
    const T *x = static_cast<const T *>(a.x) + at, *second = static_cast<const T *>(a.x2 != nullptr ? a.x2 : a.residual) + at;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool norm = !GATED && a.norm_w != nullptr;
    const int ahead = LOOSE ? static_cast<int>(at & 3) : 0;  // columns between the grid's line and the row's first
    auto column = [&](int i) { return (static_cast<int>(threadIdx.x) + i * THREADS) * 4 - ahead; };
    auto in = [&](int c) { return !LOOSE || (c >= 0 && c < a.cols); };
    auto whole = [&](int i) { return !LOOSE || (column(i) >= 0 && column(i) + 4 <= a.cols); };
    auto fetch = [&](auto &kept, const T *from, int i) {
        if (whole(i)) {
            kept.fetch(from + column(i));
        } else {
            float e[4];
#pragma unroll
            for (int l = 0; l < 4; ++l) e[l] = in(column(i) + l) ? as_float(from[column(i) + l]) : 0.0f;
            kept.keep(e);
        }
    };
    auto weights = [&](int c, float (&g)[4]) {
        if (!LOOSE) {
            load4(a.norm_w + c, g);
        } else {
#pragma unroll
            for (int l = 0; l < 4; ++l) g[l] = in(c + l) ? a.norm_w[c + l] : 0.0f;
        }
    };
    if (threadIdx.x == 0) s.largest = 0;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    Kept<T, GATED> v[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const float none[4] = {};
        if (column(i) < a.cols) fetch(v[i], x, i);
        else v[i].keep(none);
    }
    float top = 0.0f, lowest = 0.0f;
    if (GATED || a.residual != nullptr) {
        Kept<T, false> y[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (column(i) < a.cols) fetch(y[i], second, i);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (column(i) >= a.cols) continue;
            if constexpr (GATED) {
                float e[4], d[4];
                v[i].values(e);
                y[i].values(d);
                const float least = fminf(fminf(e[0], e[1]), fminf(e[2], e[3]));
                lowest = fminf(lowest, least);
                if (least < -80.0f) {
#pragma unroll
                    for (int l = 0; l < 4; ++l)  // silu(-inf) is undefined; silu(-80) = -1e-33 may have lost digits, which shows if y is large: not this way
                        if (e[l] < -80.0f && (fabsf(d[l]) > 1e3f || e[l] == -INFINITY)) top = INFINITY;
                }
#pragma unroll
                for (int l = 0; l < 4; ++l) e[l] = e[l] * d[l] * sigmoid(e[l]);  // (x y first: the product of a tiny x with the sigmoid would lose digits)
                v[i].keep(e);
            } else {
                v[i].add(y[i]);
                T *const to = static_cast<T *>(a.total) + at + column(i);
                if (whole(i)) {
                    v[i].put_to(to);
                } else {
                    float e[4];
                    v[i].values(e);
#pragma unroll
                    for (int l = 0; l < 4; ++l)
                        if (in(column(i) + l)) put(to + l, e[l]);
                }
            }
        }
    }
    double sum = 0.0;
    float best = -1.0f;  // the thread's largest product with the norm's weights, the vector it is in, whether it is there twice
    int best_at = 0;
    bool twice = false;
    if (norm) {
        double part[2] = {};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (column(i) >= a.cols) continue;
            float g[4], e[4];
            weights(column(i), g);
            v[i].values(e);
#pragma unroll
            for (int l = 0; l < 4; ++l) {
                const double d = static_cast<double>(e[l]);
                part[l & 1] = fma(d, d, part[l & 1]);
                g[l] = fabsf(e[l] * g[l]);
            }
            float most = g[0];
#pragma unroll
            for (int l = 1; l < 4; ++l) most = largest_of(most, g[l]);
            top = largest_of(top, most);
            if (most > best) best = most, best_at = i, twice = false;
            else if (most == best) twice = true;
        }
        sum = part[0] + part[1];
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float e[4];
            v[i].values(e);
#pragma unroll
            for (int l = 0; l < 4; ++l) top = largest_of(top, fabsf(e[l]));
        }
    }
    const float own = top;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = largest_of(top, __shfl_xor_sync(0xffffffffu, top, off));
    if (lane == 0) s.d[warp] = sum, s.a[warp] = top;
    __syncthreads();
    top = lane < WARPS ? s.a[lane] : 0.0f;
#pragma unroll
    for (int off = WARPS > 16 ? 16 : WARPS / 2; off > 0; off >>= 1) top = largest_of(top, __shfl_xor_sync(0xffffffffu, top, off));
    top = __shfl_sync(0xffffffffu, top, 0);
    if (!(top > (GATED ? 1e-20f : 1e-30f) && top < 1e30f)) {  // (the same in every thread: zero, tiny, huge, undefined)
        exact_row<T>(a, row, true, s);
        return;
    }
    // The largest in 64 bits.  Rounding keeps the order: of products with the norm's weights it is one whose rounded value is the largest.  Gated
    // values are off by 8e-6 at most (x = -80), so it is one within 2e-5 of it.
    if (GATED || norm) {
        const float least = GATED ? top * (1.0f - 2e-5f) : top;
        auto offer = [&](double d) { atomicMax(&s.largest, static_cast<unsigned long long>(__double_as_longlong(fabs(d)))); };
        if (own >= least && norm && !twice) {
            // (one thread, for which all the others wait: it looks at one vector only)
            const int c = column(best_at);
            float e[4], g[4];
            Kept<T, false> again;
            fetch(again, a.residual != nullptr ? static_cast<const T *>(a.total) + at : x, best_at);
            again.values(e);
            weights(c, g);
#pragma unroll
            for (int l = 0; l < 4; ++l)
                if (fabsf(e[l] * g[l]) >= least) offer(static_cast<double>(e[l]) * static_cast<double>(g[l]));
        } else if (own >= least) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (column(i) >= a.cols) continue;
                float g[4], e[4];
#pragma unroll
                for (int l = 0; l < 4; ++l) g[l] = 1.0f;
                if (norm) weights(column(i), g);
                v[i].values(e);
#pragma unroll
                for (int l = 0; l < 4; ++l)
                    if (fabsf(e[l] * g[l]) >= least)
                        offer(GATED ? exact_gate(as_float(x[column(i) + l]), as_float(second[column(i) + l])) : static_cast<double>(e[l]) * static_cast<double>(g[l]));
            }
        }
    }
    // One thread does what is left in 64 bits: that pipe is shared by the warps of all rows on the SM.
    double r = 1.0;
    if (norm && warp == 0) {
        sum = lane < WARPS ? s.d[lane] : 0.0;
#pragma unroll
        for (int off = WARPS > 16 ? 16 : WARPS / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        r = inverse_root(fma(sum, a.inv_cols, static_cast<double>(a.eps)));
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        const double largest = GATED || norm ? __longlong_as_double(static_cast<long long>(s.largest)) : static_cast<double>(top);
        const double wide = norm ? largest * r * (1.0 / 127.0) : largest / 127.0;
        const float scale = wide >= kMostScale ? kUndefined : static_cast<float>(wide);
        s.r = r;
        s.scale = static_cast<double>(scale);
        s.factor = scale > 1e-37f && r > 1.2e-38 && r < 1e38 ? __fdiv_rn(static_cast<float>(r), scale) : 0.0f;  // (r as a normal fp32 number)
        a.scales[row] = scale;
    }
    __syncthreads();
    const float f = s.factor;  // about 127 / largest
    if (f == 0.0f) {  // (a norm can take the scale or its own factor out of the middle range; so can an undefined one)
        exact_row<T>(a, row, true, s);
        return;
    }

    // To whole numbers: the sum with 1.5 * 2^23 rounds to the nearest, and holds it in its last bits.  Whoever is so near to a half that fp32 leaves it
    // open (kI8Off) is worked out in 64 bits.
    constexpr float kWhole = 12582912.0f;
    const float off = GATED ? fmaf(fmaxf(lowest, -80.0f), -kI8GatedOffPerX, kI8GatedOff) : kI8Off;
    const long long pitch = i8_pitch(a.cols);
    int8_t *out = a.q + row * pitch;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (column(i) >= a.cols) continue;
        float g[4], t[4], e[4];
        if (norm) weights(column(i), g);
        v[i].values(e);
        uint32_t bits[4];
        bool near = false;
#pragma unroll
        for (int l = 0; l < 4; ++l) {
            t[l] = (norm ? e[l] * g[l] : e[l]) * f;  // |t| < 127.1
            const float k = t[l] + kWhole;
            bits[l] = __float_as_uint(k);
            const float sure = fmaf(fabsf(t[l]), -off, 0.5f);
            t[l] = fabsf(t[l] - (k - kWhole)) - sure;
            near |= t[l] > 0.0f;
        }
        if (near) {
#pragma unroll
            for (int l = 0; l < 4; ++l)
                if (t[l] > 0.0f) {
                    double d = static_cast<double>(e[l]);
                    if (GATED) d = exact_gate(as_float(x[column(i) + l]), as_float(second[column(i) + l]));
                    else if (norm) d *= static_cast<double>(g[l]);
                    bits[l] = static_cast<uint32_t>(exact_whole(d, s.r, s.scale));
                }
        }
        if (!LOOSE) {
            *reinterpret_cast<uint32_t *>(out + column(i)) = __byte_perm(__byte_perm(bits[0], bits[1], 0x0040), __byte_perm(bits[2], bits[3], 0x0040), 0x5410);
        } else {
#pragma unroll
            for (int l = 0; l < 4; ++l)
                if (in(column(i) + l)) out[column(i) + l] = static_cast<int8_t>(bits[l]);
        }
    }
    if (threadIdx.x < pitch - a.cols) out[a.cols + threadIdx.x] = 0;
}

// (`overlap` is not among the kernel's parameters: with 8 bytes more of them 4001 rows of 5120 in fp16 take 34.2 instead of 33.6 us)
struct Place {
    bool overlap;
    int sm_count;
    cudaStream_t stream;
};

template <typename K>
cudaError_t launch_kernel(K kernel, const RowsI8Args &a, int threads, const Place &at) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3(static_cast<unsigned>(a.ntok));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.stream = at.stream;
    cfg.attrs = attr;
    cfg.numAttrs = launch_attributes(attr, at.overlap, 0);
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <typename T, int NV, int THREADS, bool LOOSE>
cudaError_t launch_variant(const RowsI8Args &a, const Place &at) {
    return a.x2 != nullptr ? launch_kernel(rows_i8_kernel<T, NV, THREADS, true, LOOSE>, a, THREADS, at)
                           : launch_kernel(rows_i8_kernel<T, NV, THREADS, false, LOOSE>, a, THREADS, at);
}
// Threads of a row: many rows have an SM to share, few rows wait for their own steps only (4 gated rows of 17408: 512 threads 6.2 us, 1024 5.2).  fp32
// rows of more than 12282 values fit twice on an SM only with spills (47 us for 40 with 512 threads each), so they take one block of 1024 (1000 gated rows of
// 17408: 52.7 us with one block of 512, 48.5).  fp16 rows of 4097 to 6138 values: 128 threads 36.1, 256 39.3 us.
// The smallest of the given numbers of vectors per thread that holds a row.
template <typename T, int THREADS, bool LOOSE, int NV, int... MORE>
cudaError_t launch_vectors(const RowsI8Args &a, const Place &at) {
    if constexpr (sizeof...(MORE) > 0)
        if ((a.cols + (LOOSE ? 6 : 3)) / 4 > NV * THREADS) return launch_vectors<T, THREADS, LOOSE, MORE...>(a, at);
    return launch_variant<T, NV, THREADS, LOOSE>(a, at);
}

template <typename T, bool LOOSE>
cudaError_t launch_size(const RowsI8Args &a, const Place &at) {
    if (a.ntok <= at.sm_count)  // few rows: as many threads on each as there are
        return a.cols <= 10234 ? launch_vectors<T, 512, LOOSE, 2, 5>(a, at) : launch_vectors<T, 1024, LOOSE, 5, 6>(a, at);
    constexpr int kMore = LOOSE ? 6 : 0;  // columns that a row may need room for, because it does not begin with a vector
    if (a.cols <= 1024 - kMore) return launch_vectors<T, 32, LOOSE, 2, 5, 8>(a, at);
    if constexpr (sizeof(T) == 2) {
        if (a.cols <= 6138) return launch_vectors<T, 128, LOOSE, 5, 8, 10, 12>(a, at);
        if (a.cols <= 12282) return launch_vectors<T, 256, LOOSE, 8, 10, 12>(a, at);
        return launch_vectors<T, 512, LOOSE, 8, 9, 10, 12>(a, at);
    } else {
        if (a.cols <= 4096 - kMore) return launch_vectors<T, 128, LOOSE, 5, 8>(a, at);
        if (a.cols <= 12282) return launch_vectors<T, 256, LOOSE, 5, 8, 10, 12>(a, at);
        return launch_vectors<T, 1024, LOOSE, 5, 6>(a, at);
    }
}
template <typename T>
cudaError_t launch_t(const RowsI8Args &a, const Place &at) {
    if (a.x2 != nullptr && a.norm_w != nullptr && i8_pitch(a.cols) <= 512 * 40) {
        if (i8_pitch(a.cols) <= 512 * 4) return launch_kernel(gated_norm_kernel<T, 4>, a, 512, at);
        if (i8_pitch(a.cols) <= 512 * 16) return launch_kernel(gated_norm_kernel<T, 16>, a, 512, at);
        return launch_kernel(gated_norm_kernel<T, 40>, a, 512, at);
    }
    if (a.cols > kMostFast || (a.x2 != nullptr && a.norm_w != nullptr)) return launch_kernel(exact_rows_kernel<T>, a, 512, at);
    return a.cols % 4 == 0 ? launch_size<T, false>(a, at) : launch_size<T, true>(a, at);
}

}  // namespace

cudaError_t launch_rows_i8(const RowsI8Args &in, bool overlap, int sm_count, cudaStream_t stream) {
    RowsI8Args a = in;
    a.inv_cols = 1.0 / a.cols;
    const Place at{overlap, sm_count, stream};
    return a.elem == 2 ? launch_t<__half>(a, at) : launch_t<float>(a, at);
}

}  // namespace vqm
