// Two fp32 in one instruction (vqm_rows_f8.cu, vqm_logprobs.cu).
#pragma once

namespace vqm {
namespace {

using Two = unsigned long long;
__device__ __forceinline__ Two two(float x, float y) {
    Two v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
    return v;
}
__device__ __forceinline__ void both(Two v, float &x, float &y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ Two add2(Two a, Two b) {
    Two v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
    Two v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
    Two v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}

}  // namespace
}  // namespace vqm
