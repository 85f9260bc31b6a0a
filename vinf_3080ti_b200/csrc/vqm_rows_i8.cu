// Activation rows as 8-bit integers with a scale per row, after what a layer does to them on the way to a projection:
//   v = x,  or silu(x) * x2,  or h = x + residual (rounded to its type and stored);   n = v * g / sqrt(mean(v^2) + eps), or v;
//   s = max |n| / 127 in fp32,   q = n / s rounded to the nearest whole number, ties to even.
// All of it is done in 64 bits: which of two whole numbers a value goes to is then decided by the formula, not by the order of 32-bit
// roundings.
#include <cuda_fp16.h>

#include "vqm_kernels.h"

namespace vqm {
namespace {

constexpr int kRowThreads = 512;

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ void put(float *p, float v) { *p = v; }
__device__ __forceinline__ void put(__half *p, float v) { *p = __float2half_rn(v); }

template <typename T>
__global__ void __launch_bounds__(kRowThreads) rows_i8_kernel(const RowsI8Args a) {
    __shared__ double s_red[kRowThreads / 32];
    __shared__ int s_bad;
    const size_t row = blockIdx.x, at = row * a.cols;
    const T *x = static_cast<const T *>(a.x) + at, *x2 = static_cast<const T *>(a.x2) + at, *res = static_cast<const T *>(a.residual) + at;
    T *total = static_cast<T *>(a.total) + at;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto value = [&](int c) -> double {
        if (a.residual != nullptr) return as_float(total[c]);  // (by the thread that wrote it)
        const double v = as_float(x[c]);
        return a.x2 != nullptr ? v / (1.0 + exp(-v)) * static_cast<double>(as_float(x2[c])) : v;
    };
    auto combine = [&](double v, auto op) -> double {
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, off));
        __syncthreads();
        if (lane == 0) s_red[warp] = v;
        __syncthreads();
        v = s_red[0];
        for (int i = 1; i < kRowThreads / 32; ++i) v = op(v, s_red[i]);
        return v;
    };
    if (a.residual != nullptr)
        for (int c = threadIdx.x; c < a.cols; c += kRowThreads) put(total + c, as_float(x[c]) + as_float(res[c]));
    double r = 1.0;
    if (a.norm_w != nullptr) {
        double sum = 0.0;
        for (int c = threadIdx.x; c < a.cols; c += kRowThreads) {
            const double v = value(c);
            sum += v * v;
        }
        sum = combine(sum, [](double p, double q) { return p + q; });
        r = 1.0 / sqrt(sum / a.cols + static_cast<double>(a.eps));
    }
    if (threadIdx.x == 0) s_bad = 0;
    double top = 0.0;
    bool bad = false;
    for (int c = threadIdx.x; c < a.cols; c += kRowThreads) {
        const double n = a.norm_w != nullptr ? value(c) * r * static_cast<double>(a.norm_w[c]) : value(c);
        bad |= !(fabs(n) <= 1e300);
        top = fmax(top, fabs(n));
    }
    top = combine(top, [](double p, double q) { return fmax(p, q); });
    if (bad) s_bad = 1;
    __syncthreads();
    float s = static_cast<float>(top / 127.0);
    // a value that is infinite or undefined makes the row's outputs undefined
    if (s_bad || !(s <= 3.4028235e38f)) s = __int_as_float(0x7fc00000);
    if (threadIdx.x == 0) a.scales[row] = s;
    const long long pitch = i8_pitch(a.cols);
    for (int c = threadIdx.x; c < pitch; c += kRowThreads) {
        int q = 0;
        if (c < a.cols && s > 0.0f) {
            const double n = a.norm_w != nullptr ? value(c) * r * static_cast<double>(a.norm_w[c]) : value(c);
            q = min(127, max(-127, __double2int_rn(n / static_cast<double>(s))));
        }
        a.q[row * pitch + c] = static_cast<int8_t>(q);
    }
}

}  // namespace

cudaError_t launch_rows_i8(const RowsI8Args &a, cudaStream_t stream) {
    if (a.elem == 2) rows_i8_kernel<__half><<<a.ntok, kRowThreads, 0, stream>>>(a);
    else rows_i8_kernel<float><<<a.ntok, kRowThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace vqm
