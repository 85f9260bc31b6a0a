// Verification of drafted tokens.  Draft i of a sequence, drawn from q_i = softmax(draft logits / T), is accepted if
// u_i q_i(token) < p_i(token) with p_i = softmax(target logits / T); after the first refusal, or behind the last draft, one more token is
// drawn from max(p - q, 0) (or from p) by inverse cdf with the last random number.  That the tokens are distributed as the target's
// own holds for any q; a draft without probabilities is q = 1 at its token.
#include <cuda_fp16.h>

#include "vqm_kernels.h"

namespace vqm {
namespace {

constexpr int kVerifyThreads = 1024, kVerifyWarps = kVerifyThreads / 32;

__device__ __forceinline__ float logit(const float *p) { return *p; }
__device__ __forceinline__ float logit(const __half *p) { return __half2float(*p); }

// A row's probabilities: weight(i) / sum.
template <typename T>
struct Row {
    const T *x;
    double top, scale, sum;  // largest logit, 1 / T (negative: greedy), sum of the weights
    int first;               // lowest index of the largest logit
    __device__ double weight(int i) const {
        const float v = logit(x + i);
        if (!(v > -INFINITY)) return 0.0;
        if (scale < 0.0) return i == first ? 1.0 : 0.0;
        return v == static_cast<float>(top) ? 1.0 : exp((static_cast<double>(v) - top) * scale);
    }
    __device__ double p(int i) const { return sum > 0.0 ? weight(i) / sum : 0.0; }
};

struct Shared {
    double d[kVerifyWarps];
    float f[kVerifyWarps];
    int i[kVerifyWarps];
};

__device__ double block_sum(double v, Shared &s) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.d[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < kVerifyWarps; ++w) v += s.d[w];
    return v;
}

template <typename T>
__device__ Row<T> look(const T *x, int n, float temperature, Shared &s) {
    float top = -INFINITY;
    int first = n;
    for (int i = threadIdx.x; i < n; i += kVerifyThreads) {
        const float v = logit(x + i);
        if (v > top) top = v, first = i;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        const float v = __shfl_xor_sync(0xffffffffu, top, off);
        const int j = __shfl_xor_sync(0xffffffffu, first, off);
        if (v > top || (v == top && j < first)) top = v, first = j;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.f[threadIdx.x >> 5] = top, s.i[threadIdx.x >> 5] = first;
    __syncthreads();
    top = s.f[0], first = s.i[0];
    for (int w = 1; w < kVerifyWarps; ++w)
        if (s.f[w] > top || (s.f[w] == top && s.i[w] < first)) top = s.f[w], first = s.i[w];
    Row<T> row{x, static_cast<double>(top), temperature > 0.0f ? fmax(1.0 / static_cast<double>(temperature), 1e-300) : -1.0, 0.0, first};
    double sum = 0.0;
    for (int i = threadIdx.x; i < n; i += kVerifyThreads) sum += row.weight(i);
    row.sum = block_sum(sum, s);
    return row;
}

template <typename T>
__global__ void __launch_bounds__(kVerifyThreads) verify_kernel(const VerifyArgs a) {
    __shared__ Shared s;
    const int seq = blockIdx.x, k = a.drafts, n = a.vocab;
    const float temperature = a.temperature != nullptr ? a.temperature[seq] : 1.0f;
    const float *u = a.uniforms + static_cast<size_t>(seq) * (k + 1);
    int *out = a.out + static_cast<size_t>(seq) * (k + 2);
    const int len = a.lens != nullptr ? min(k, max(0, a.lens[seq])) : k;
    const T *target = static_cast<const T *>(a.target) + static_cast<size_t>(seq) * (k + 1) * n;
    const T *draft = static_cast<const T *>(a.draft) + static_cast<size_t>(seq) * k * n;
    int j = 0, token = -1;
    Row<T> p{}, q{};
    for (;; ++j) {
        p = look(target + static_cast<size_t>(j) * n, n, temperature, s);
        if (j == len) break;
        token = a.tokens[static_cast<size_t>(seq) * k + j];
        if (a.draft != nullptr) q = look(draft + static_cast<size_t>(j) * n, n, temperature, s);
        if (token < 0 || token >= n) break;  // no token: refused
        const double qt = a.draft != nullptr ? q.p(token) : 1.0;
        if (!(static_cast<double>(u[j]) * qt < p.p(token))) break;
        if (threadIdx.x == 0) out[1 + j] = token;
    }
    // the token behind: weights r(i), smallest i whose sum up to it is above u times the whole
    bool minus = j < len;
    auto rest = [&](int i) -> double {
        const double pi = p.p(i);
        if (!minus) return pi;
        const double d = pi - (a.draft != nullptr ? q.p(i) : i == token ? 1.0 : 0.0);
        return d > 0.0 ? d : 0.0;
    };
    double mine = 0.0;
    const int per = (n + kVerifyThreads - 1) / kVerifyThreads, i0 = min(n, static_cast<int>(threadIdx.x) * per), i1 = min(n, i0 + per);
    for (int i = i0; i < i1; ++i) mine += rest(i);
    double whole = block_sum(mine, s);
    if (minus && !(whole > 0.0)) {
        minus = false;
        mine = 0.0;
        for (int i = i0; i < i1; ++i) mine += rest(i);
        whole = block_sum(mine, s);
    }
    __shared__ double s_part[kVerifyThreads];
    s_part[threadIdx.x] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
        int next = -1;
        if (whole > 0.0) {
            const double point = static_cast<double>(u[k]) * whole;
            double sum = 0.0;
            int last = -1;  // the last part with a weight
            int found = -1;
            for (int t = 0; t < kVerifyThreads; ++t) {
                if (s_part[t] > 0.0) last = t;
                if (sum + s_part[t] > point) {
                    found = t;
                    break;
                }
                sum += s_part[t];
            }
            if (found < 0) found = last;
            for (int i = min(n, found * per); i < min(n, found * per + per); ++i) {
                const double r = rest(i);
                if (r > 0.0) next = i;
                sum += r;
                if (r > 0.0 && sum > point) break;
            }
        }
        out[0] = j;
        out[1 + j] = next;
        for (int i = j + 2; i < k + 2; ++i) out[i] = -1;
    }
}

}  // namespace

cudaError_t launch_verify(const VerifyArgs &a, int sm_count, cudaStream_t stream) {
    (void)sm_count;
    if (a.elem == 2) verify_kernel<__half><<<a.seqs, kVerifyThreads, 0, stream>>>(a);
    else verify_kernel<float><<<a.seqs, kVerifyThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace vqm
