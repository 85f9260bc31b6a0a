// Log probabilities of given tokens, the entropy of the distribution they are drawn from, and its likeliest tokens:  p = softmax(l / T),
//   out = log p(token),   entropy = - sum p log p,   the `top` largest logits, of equal ones the lowest place first.
// Simple form: a block of threads per row; a pass for the largest logit, one for the sums in 64 bits, one for each alternative.
#include <cuda_fp16.h>

#include "vqm_kernels.h"

namespace vqm {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }

// A logit and its place as one number, larger for what comes first: by value, then by the lower place.  0: nothing (masked).
__device__ __forceinline__ unsigned long long key_of(float v, int i) {
    if (!(v > -INFINITY)) return 0;
    const uint32_t b = __float_as_uint(v == 0.0f ? 0.0f : v);  // (the zeros are equal)
    return static_cast<unsigned long long>((b & 0x80000000u) != 0 ? ~b : b | 0x80000000u) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(i));
}
__device__ __forceinline__ int place_of(unsigned long long key) { return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(key)); }

template <typename V, typename F>
__device__ V over_block(V v, V (&room)[kWarps], F &&join) {
    for (int off = 16; off > 0; off >>= 1) v = join(v, __shfl_xor_sync(0xFFFFFFFFu, v, off));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) room[threadIdx.x >> 5] = v;
    __syncthreads();
    v = room[0];
    for (int w = 1; w < kWarps; ++w) v = join(v, room[w]);
    return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(const LogprobsArgs a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ double s_sum[kWarps];
    __shared__ unsigned long long s_key[kWarps];
    const size_t row = blockIdx.x;
    const T *x = static_cast<const T *>(a.logits) + row * a.vocab;
    const float given = a.temperature != nullptr ? a.temperature[row] : 1.0f;
    const bool greedy = !(given > 0.0f), broken = *a.status != 0;
    auto larger = [](unsigned long long p, unsigned long long q) { return p > q ? p : q; };
    auto plus = [](double p, double q) { return p + q; };
    auto next = [&](unsigned long long below) {  // the largest key under that
        unsigned long long most = 0;
        for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
            const unsigned long long k = key_of(as_float(x[i]), i);
            if (k < below && k > most) most = k;
        }
        return over_block(most, s_key, larger);
    };
    const unsigned long long first = next(~0ull);
    const float top = first != 0 ? as_float(x[place_of(first)]) : 0.0f;
    const bool flat = given > 1e30f && top < INFINITY;
    const double inv = 1.0 / static_cast<double>(given);
    auto less = [&](float v, int i) -> double {  // (logit - largest) / T, -inf where p is nothing
        if (!(v > -INFINITY)) return -INFINITY;
        if (greedy) return i == place_of(first) ? 0.0 : -INFINITY;
        if (v == top || flat) return 0.0;
        return top == INFINITY ? -INFINITY : (static_cast<double>(v) - static_cast<double>(top)) * inv;
    };
    double sum = 0.0, weighted = 0.0;
    for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
        const double d = less(as_float(x[i]), i), e = exp(d);
        sum += e;
        if (e > 0.0) weighted -= e * d;
    }
    sum = over_block(sum, s_sum, plus);
    weighted = over_block(weighted, s_sum, plus);
    const double log_sum = sum > 0.0 ? log(sum) : 0.0;
    auto answer = [&](float v, int i) { return broken ? __uint_as_float(0x7FFFFFFFu) : static_cast<float>(less(v, i) - log_sum); };
    if (threadIdx.x == 0) {
        const int token = a.tokens[row];
        const bool inside = token >= 0 && token < a.vocab;
        a.out[row] = answer(inside ? as_float(x[token]) : -INFINITY, token);
        if (a.entropy != nullptr) a.entropy[row] = broken ? __uint_as_float(0x7FFFFFFFu) : sum > 0.0 ? static_cast<float>(log_sum + weighted / sum) : 0.0f;
    }
    unsigned long long k = first;
    for (int j = 0; j < a.top; ++j) {
        if (threadIdx.x == 0) {
            const size_t to = row * a.top + j;
            a.top_ids[to] = k != 0 && !broken ? place_of(k) : -1;
            if (a.top_out != nullptr) a.top_out[to] = answer(k != 0 ? as_float(x[place_of(k)]) : -INFINITY, place_of(k));
        }
        if (k != 0 && j + 1 < a.top) k = next(k);
    }
}

}  // namespace

cudaError_t launch_logprobs(const LogprobsArgs &a, bool overlap, int sm_count, cudaStream_t stream) {
    (void)sm_count;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[2];
    cfg.gridDim = dim3(static_cast<unsigned>(a.rows));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = launch_attributes(attr, overlap, 0);
    return a.elem == 2 ? cudaLaunchKernelEx(&cfg, logprobs_kernel<__half>, a) : cudaLaunchKernelEx(&cfg, logprobs_kernel<float>, a);
}

}  // namespace vqm
