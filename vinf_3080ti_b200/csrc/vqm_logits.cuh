// Rows of logits in vectors of 16 bytes, wherever they begin (vqm_verify.cu, vqm_logprobs.cu).
#pragma once

#include <cuda_fp16.h>

#include <cstdint>

namespace vqm {
namespace {

template <typename T>
constexpr int kVec = 16 / static_cast<int>(sizeof(T));

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }

// 16 bytes of a row, vector `v` of its 16-byte grid; elements outside of [0, n) are -inf.  first: index of vector 0's first element (0 or negative).
// Kept as they come until they are used: half the registers for 16-bit logits.
__device__ __forceinline__ void load_vec(const float *x, int n, int first, int v, uint4 &out) {
    const int i = first + v * 4;
    if (i >= 0 && i + 4 <= n) {
        out = *reinterpret_cast<const uint4 *>(x + i);
    } else {
        uint32_t r[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = __float_as_uint(i + e >= 0 && i + e < n ? x[i + e] : -INFINITY);
        out = make_uint4(r[0], r[1], r[2], r[3]);
    }
}
__device__ __forceinline__ void load_vec(const __half *x, int n, int first, int v, uint4 &out) {
    const int i = first + v * 8;
    if (i >= 0 && i + 8 <= n) {
        out = *reinterpret_cast<const uint4 *>(x + i);
    } else {
        uint32_t r[4] = {};
#pragma unroll
        for (int e = 0; e < 8; ++e)
            r[e / 2] |= (i + e >= 0 && i + e < n ? static_cast<uint32_t>(__half_as_ushort(x[i + e])) : 0xFC00u) << (16 * (e & 1));
        out = make_uint4(r[0], r[1], r[2], r[3]);
    }
}
__device__ __forceinline__ void values_of(const uint4 &w, float (&out)[4]) {
    out[0] = __uint_as_float(w.x), out[1] = __uint_as_float(w.y), out[2] = __uint_as_float(w.z), out[3] = __uint_as_float(w.w);
}
__device__ __forceinline__ void values_of(const uint4 &w, float (&out)[8]) {
    const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&r[e]));
        out[2 * e] = f.x, out[2 * e + 1] = f.y;
    }
}
template <typename T>
constexpr uint32_t kNothing = sizeof(T) == 4 ? 0xFF800000u : 0xFC00FC00u;  // -inf
template <typename T>
__device__ __forceinline__ int first_of(const T *x) {  // index of the first element of the row's first aligned vector
    return -static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

}  // namespace
}  // namespace vqm
