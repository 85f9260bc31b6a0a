// Verification of drafted tokens.  Draft i of a sequence, drawn from q_i = softmax(draft logits / T), is accepted if
// u_i q_i(token) < p_i(token) with p_i = softmax(target logits / T); after the first refusal, or behind the last draft, one more token is
// drawn from max(p - q, 0) (or from p) by inverse cdf with the last random number.  That the tokens are distributed as the target's
// own holds for any q; a draft without probabilities is q = 1 at its token.
//
// One cluster per sequence, each block a slice of the vocabulary.
//   1. One pass over the logits: every row's largest and the sum of exp over it, in fp32 (exponentials by ex2, sums of at most some hundred terms
//      per lane).  The blocks exchange (largest, sum) of each row through distributed shared memory.
//   2. Every block decides on all drafts.  fp32 leaves the two sides of a test uncertain by about 1e-6; where they are within 1e-4 of one another, and for rows
//      with values that fp32 cannot hold (infinite, undefined, too large over T), the cluster sums the row's exponentials again in 64 bits.
//   3. The token behind: which of 150000 intervals the random number falls into hangs on the 12th digit of the sums, so the one or two rows it
//      takes are summed in 64 bits: both rows' sums, then the weights by blocks and warps, then within one warp's part.
// Nothing is kept in device memory between the steps: launches on several streams and in several graphs do not meet.
//
// What bounds it: 64 sequences x 4 drafts x 151936 in fp32 take 157 us of one stream (2230 GB/s; three streams: 84 us a call, 4150 GB/s): 60 us are step 1, near
// the copy bandwidth, the rest the exponentials in 64 bits of two rows (eight instructions of that pipe and some twenty others each: 45 cycles per 32 of them
// and scheduler, whatever of loads, table or series is left out).  One sequence x 3 drafts: 31 us on 16 SMs, as many as a cluster takes.  Of that, half
// is the steps' latency: a vocabulary of 1000 takes 16 us.  Tried: 1024 threads, two blocks of 256 or 512 per SM (spills), a second round of
// clusters, both rows' weights kept in shared memory between their two passes (no gain).
#include <cuda_fp16.h>

#include "vqm_kernels.h"
#include "vqm_tcmv.cuh"

namespace vqm {
namespace {

constexpr int kVThreads = 512, kVWarps = kVThreads / 32, kVMaxCluster = 16, kVMaxRows = 2 * 255 + 1;
constexpr int kVTable = 128, kVCopies = 16;  // entries of 2^(j / 128), and copies: lanes that look up at random do not meet in a bank
constexpr double kVMagic = 6755399441055744.0 / kVTable;  // 1.5 * 2^52 / 128: adding it rounds to a multiple of 1 / 128
constexpr double kNoise = 1.0 / (1ull << 44);  // p - q within the rounding of the rows' sums is nothing: equal rows leave no rest
constexpr double kLn2 = 0.693147180559945309417232121458, kLog2e = 1.0 / kLn2;

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
__device__ __forceinline__ float cluster_load(uint32_t at) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ double cluster_load_double(uint32_t at) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(at) : "memory");
    return v;
}

constexpr int kNoIndex = 0x7fffffff;
struct Shared {
    double table[kVTable][kVCopies];
    float part_top[kVMaxRows + kVWarps], part_sum[kVMaxRows + kVWarps];  // the warps', by row + warp (rows: target 0, draft 0, target 1, ...)
    float top[kVMaxRows], sum[kVMaxRows];          // this block's (greedy: lowest index of the largest, as int bits)
    float all_top[kVMaxRows], all_sum[kVMaxRows];  // the whole row's
    unsigned char verdict[256];                    // of the drafts
    double warp_sum[2][kVWarps];                // of the warps; of the row(s) being summed
    double block_sum[2][2];                        // this block's, for the others; two buffers in turn
};
enum : unsigned char { kAccept, kRefuse, kUnsure };

// A row's weights exp((x - top) / T) in 64 bits, all of them times one factor near 1: 2^(x log2(e) / T - shift) with a shift that is a multiple of 1 / 128.
struct Weights {
    double scale, magic;  // log2(e) / T, kVMagic - shift
    float least;          // a smaller logit weighs 2^-1000, which counts as nothing (and so does a masked or undefined one)
    bool plain;           // everything above is within its bounds
    float top;
    double inv_t;
};
constexpr double kTiny = 0x1p-960;

// 2^y with y = x scale - shift: y = j / 128 + r, |r| <= 1 / 256; 2^(j / 128) by table, 2^r by the series of exp up to the fourth power of
// r ln 2 < 0.00271, which leaves 1.2e-15 (table-driven exponential: P. Tang, ACM TOMS 15, 1989).  Eight instructions of the 64-bit pipe.
template <int N>
__device__ __forceinline__ void powers(const float *x, const Weights &w, const double *table, double *out) {
    double t[N], r[N], f[N];
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = static_cast<double>(fmaxf(x[i], w.least));
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = fma(out[i], w.scale, w.magic);  // kVMagic + j / 128
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int n = __double2loint(t[i]);
        const double two = table[(n & (kVTable - 1)) * kVCopies];
        f[i] = __hiloint2double(__double2hiint(two) + (n & -kVTable) * ((1 << 20) / kVTable), __double2loint(two));
        r[i] = fma(out[i], w.scale, w.magic - t[i]);  // (the difference is exact)
    }
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = fma(r[i], kLn2 * kLn2 * kLn2 * kLn2 / 24.0, kLn2 * kLn2 * kLn2 / 6.0);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = fma(out[i], r[i], kLn2 * kLn2 / 2.0);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = fma(out[i], r[i], kLn2);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = fma(out[i], r[i], 1.0);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] *= f[i];
}
// Rows whose largest logit or temperature is out of the ordinary; not inlined: cold code costs every launch its fetch.
static __device__ __noinline__ double rare_weight(float x, float top, double inv_t) {
    return !(x > -INFINITY) ? 0.0 : x == top ? 1.0 : exp((static_cast<double>(x) - static_cast<double>(top)) * inv_t);
}
__device__ __forceinline__ double weight(float x, const Weights &w, const double *table) {
    double p;
    if (w.plain) powers<1>(&x, w, table, &p);
    else p = rare_weight(x, w.top, w.inv_t);
    return p > kTiny ? p : 0.0;
}
__device__ __forceinline__ Weights weights_of(float top, float temperature) {
    Weights w;
    w.top = top;
    w.inv_t = fmax(1.0 / static_cast<double>(temperature), 1e-300);
    w.scale = w.inv_t * kLog2e;
    const double shift = static_cast<double>(top) * w.scale;
    w.magic = kVMagic - shift;  // (rounds the shift)
    w.least = static_cast<float>(static_cast<double>(top) - 1000.0 / w.scale);
    w.plain = fabs(shift) < 1e7 && w.scale > 1e-30 && w.scale < 1e30;
    return w;
}

__device__ __forceinline__ double warp_total(double v) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}
// The one or two rows that the token behind is drawn from.
template <typename T>
struct Rest {
    const T *x, *y;      // target's and (or null) draft's
    Weights wp, wq;
    double inv_p, inv_q;  // 1 / sums
    const double *table;
    int n, first, token;  // token: drafted without probabilities, its weight is taken off (or -1)
    enum { kSums, kRise, kTarget } what;  // sums of both rows; weights max(p - q, 0); weights p

    template <bool BOTH>
    __device__ __forceinline__ void load(int v, uint4 &e, uint4 &d) const {
        load_vec(x, n, first, v, e);
        if (!BOTH || y == nullptr) return;
        if (first_of(y) == first) {
            load_vec(y, n, first, v, d);
        } else {  // the draft's row lies on another grid
            uint32_t r[4] = {};
#pragma unroll
            for (int i = 0; i < kVec<T>; ++i) {
                const int at = first + v * kVec<T> + i;
                const bool in = at >= 0 && at < n;
                if constexpr (sizeof(T) == 4) r[i] = in ? __float_as_uint(as_float(y[at])) : kNothing<T>;
                else r[i / 2] |= (in ? static_cast<uint32_t>(__half_as_ushort(y[at])) : 0xFC00u) << (16 * (i & 1));
            }
            d = make_uint4(r[0], r[1], r[2], r[3]);
        }
    }
    __device__ __forceinline__ double of(float e, float d, int at) const {
        const double p = weight(e, wp, table);
        if (what == kTarget) return at == token ? 0.0 : p;
        const double a = __dmul_rn(p, inv_p), rise = a - __dmul_rn(weight(d, wq, table), inv_q);
        return rise > a * kNoise ? rise : 0.0;
    }
    // this warp's sums over vectors [v0, v1), in every lane
    __device__ __noinline__ double2 sums(int v0, int v1) const {
        if (!wp.plain || !wq.plain) return rare_sums(v0, v1);
        return what == kRise ? plain_sums<true, true>(v0, v1) : y != nullptr && what == kSums ? plain_sums<true, false>(v0, v1) : plain_sums<false, false>(v0, v1);
    }
    template <bool BOTH, bool RISE>
    __device__ __forceinline__ double2 plain_sums(int v0, int v1) const {
        double a = 0.0, b = 0.0;
        const Weights p = wp, q = wq;
        const double by_p = inv_p, by_q = inv_q;
        const double *const powers_of = table;
        const int skip = what == kTarget && token >= 0 ? token : -1;
        auto take = [&](int v, const uint4 &e_raw, const uint4 &d_raw) {
            float e[kVec<T>], d[kVec<T>];
            values_of(e_raw, e);
            if (BOTH) values_of(d_raw, d);
            if (!BOTH) {
                const unsigned at = static_cast<unsigned>(skip - (first + v * kVec<T>));
                if (at < kVec<T>) {
#pragma unroll
                    for (int l = 0; l < kVec<T>; ++l)
                        if (at == l) e[l] = -INFINITY;
                }
            }
#pragma unroll
            for (int i = 0; i < kVec<T>; i += 4) {  // four elements of one or two rows side by side
                double w[4], z[4];
                powers<4>(e + i, p, powers_of, w);
                if (BOTH) powers<4>(d + i, q, powers_of, z);
                if (RISE) {
#pragma unroll
                    for (int l = 0; l < 4; ++l) {
                        const double x = __dmul_rn(w[l], by_p), diff = x - __dmul_rn(z[l], by_q);
                        w[l] = diff > x * kNoise ? diff : 0.0;
                    }
                }
                a += (w[0] + w[1]) + (w[2] + w[3]);
                if (BOTH && !RISE) b += (z[0] + z[1]) + (z[2] + z[3]);
            }
        };
        auto fetch = [&](int v, uint4 &e, uint4 &d) {
            if (v < v1) load<BOTH>(v, e, d);
        };
        uint4 e0, d0, e1, d1;
        int v = v0 + static_cast<int>(threadIdx.x & 31);
        fetch(v, e0, d0);
        fetch(v + 32, e1, d1);
        for (; v < v1; v += 64) {  // (the next two are on their way)
            take(v, e0, d0);
            fetch(v + 64, e0, d0);
            if (v + 32 >= v1) break;
            take(v + 32, e1, d1);
            fetch(v + 96, e1, d1);
        }
        return make_double2(warp_total(a), warp_total(b));
    }
    __device__ __noinline__ double2 rare_sums(int v0, int v1) const {
        double a = 0.0, b = 0.0;
        for (int v = v0 + static_cast<int>(threadIdx.x & 31); v < v1; v += 32) {
            uint4 e_raw, d_raw = make_uint4(0, 0, 0, 0);
            load<true>(v, e_raw, d_raw);
            float e[kVec<T>], d[kVec<T>];
            values_of(e_raw, e);
            values_of(d_raw, d);
#pragma unroll 1
            for (int i = 0; i < kVec<T>; ++i) {
                const float ei = element(e, i), di = element(d, i);
                if (what == kSums) a += weight(ei, wp, table), b += y != nullptr ? weight(di, wq, table) : 0.0;
                else a += of(ei, di, first + v * kVec<T> + i);
            }
        }
        return make_double2(warp_total(a), warp_total(b));
    }
    __device__ __forceinline__ static float element(const float (&e)[kVec<T>], int i) {
        float v = e[0];
#pragma unroll
        for (int l = 1; l < kVec<T>; ++l) v = l == i ? e[l] : v;
        return v;
    }
};

template <typename T>
__global__ void __launch_bounds__(kVThreads, 1) verify_kernel(const VerifyArgs a) {
    __shared__ Shared s;
    constexpr int VEC = kVec<T>, WARPS = kVWarps;
    uint32_t n_blocks, block;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n_blocks));
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(block));
    const int seq = static_cast<int>(blockIdx.x / n_blocks), k = a.drafts, n = a.vocab, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int i = threadIdx.x; i < kVTable; i += kVThreads) {
        const double p = exp2(static_cast<double>(i) / kVTable);
        for (int l = 0; l < kVCopies; ++l) s.table[i][(i + l) % kVCopies] = p;
    }
    const double *const table = &s.table[0][lane % kVCopies];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const float temperature = a.temperature != nullptr ? a.temperature[seq] : 1.0f;
    const bool greedy = !(temperature > 0.0f);
    const float *u = a.uniforms + static_cast<size_t>(seq) * (k + 1);
    const int *tokens = a.tokens + static_cast<size_t>(seq) * k;
    int *out = a.out + static_cast<size_t>(seq) * (k + 2);
    const int len = a.lens != nullptr ? min(k, max(0, a.lens[seq])) : k;
    const bool with_draft = a.draft != nullptr && !greedy;  // (greedy verification asks for the target's largest only)
    const T *target = static_cast<const T *>(a.target) + static_cast<size_t>(seq) * (k + 1) * n;
    const T *draft = static_cast<const T *>(a.draft) + static_cast<size_t>(seq) * k * n;
    const int per_step = with_draft ? 2 : 1, n_rows = len * per_step + 1;  // row r: target r / per_step, or its draft
    auto sync_cluster = [&] {
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    };
    // Vectors [from, from + share) of every row's own 16-byte grid are this block's.
    const int share = ((n + VEC - 1) / VEC + 1 + static_cast<int>(n_blocks) - 1) / static_cast<int>(n_blocks), from = static_cast<int>(block) * share;

    // ---- 1. largest and sum of every row.  The block's shares of all rows, one behind the other, are dealt to its warps in equal parts: a
    //      warp has one or two ends of a row to reduce, and reads in between without a pause.
    const float c = static_cast<float>(kLog2e / static_cast<double>(temperature));
    const long long total = static_cast<long long>(n_rows) * share;
    // (largest, sum) of two parts; greedy: (largest, its lowest index)
    auto join = [&](float &top, float &sum, float t, float v) {
        if (greedy) {
            if (t > top || (t == top && __float_as_int(v) < __float_as_int(sum))) top = t, sum = v;
        } else {
            const float most = fmaxf(top, t);
            sum = (top == most ? sum : sum * ex2((top - most) * c)) + (t == most ? v : v * ex2((t - most) * c));
            top = most;
        }
    };
    auto join_lanes = [&](float &top, float &sum) {
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
            const float t = __shfl_xor_sync(0xffffffffu, top, off), v = __shfl_xor_sync(0xffffffffu, sum, off);
            join(top, sum, t, v);
        }
    };
    const float none = greedy ? __int_as_float(kNoIndex) : 0.0f;
    {
        long long f = total * warp / WARPS;
        const long long f_end = total * (warp + 1) / WARPS;
#pragma unroll 1
        for (int r = static_cast<int>(f / share); f < f_end; ++r) {
            const int i = with_draft ? r >> 1 : r;
            const T *x = with_draft && (r & 1) ? draft + static_cast<size_t>(i) * n : target + static_cast<size_t>(i) * n;
            const int first = first_of(x), n_vec = (n - first + VEC - 1) / VEC;
            const long long base = static_cast<long long>(r) * share;
            const int v0 = from + static_cast<int>(f - base), v1 = min(n_vec, from + static_cast<int>(min(f_end - base, static_cast<long long>(share))));
            f = base + share;
            float top = -INFINITY, sum = none;
            constexpr int U = 4;
            uint4 raw[2][U];  // what is being added up, and the next on its way
            auto fetch = [&](int v, uint4 (&to)[U]) {
#pragma unroll
                for (int j = 0; j < U; ++j) {
                    if (v + j * 32 < v1) load_vec(x, n, first, v + j * 32, to[j]);
                    else to[j] = make_uint4(kNothing<T>, kNothing<T>, kNothing<T>, kNothing<T>);
                }
            };
            auto take = [&](int v, const uint4 (&from_raw)[U]) {
                float e[U][VEC];
#pragma unroll
                for (int j = 0; j < U; ++j) values_of(from_raw[j], e[j]);
                float most = e[0][0];
#pragma unroll
                for (int j = 0; j < U; ++j)
#pragma unroll
                    for (int l = 0; l < VEC; ++l) most = fmaxf(most, e[j][l]);  // (undefined ones lose)
                if (greedy) {
                    if (most > top) {
                        top = most;
#pragma unroll
                        for (int j = U - 1; j >= 0; --j)
#pragma unroll
                            for (int l = VEC - 1; l >= 0; --l)
                                if (e[j][l] == most) sum = __int_as_float(first + (v + j * 32) * VEC + l);
                    }
                    return;
                }
                if (most > top) {
                    sum *= ex2((top - most) * c);
                    top = most;
                }
                const float base_top = top > -INFINITY ? top : 0.0f;  // (differences first: no digits of large logits are lost)
                float part[4] = {};
#pragma unroll
                for (int j = 0; j < U; ++j)
#pragma unroll
                    for (int l = 0; l < VEC; ++l) part[l & 3] += ex2((e[j][l] - base_top) * c);
                sum += (part[0] + part[1]) + (part[2] + part[3]);
            };
            int v = v0 + lane;
            fetch(v, raw[0]);
#pragma unroll 1
            for (; __any_sync(0xffffffffu, v < v1); v += 2 * U * 32) {
                fetch(v + U * 32, raw[1]);
                take(v, raw[0]);
                fetch(v + 2 * U * 32, raw[0]);
                take(v + U * 32, raw[1]);
            }
            join_lanes(top, sum);
            // (a warp's last row is at most the next one's first: row + warp is a place of its own)
            if (lane == 0) s.part_top[r + warp] = top, s.part_sum[r + warp] = sum;
        }
    }
    // what the drafts' tests need beside the sums
    int my_token = -1;
    float my_x = 0.0f, my_y = 0.0f, my_u = 0.0f;
    static_assert(kVThreads >= 256, "a thread per draft");
    if (static_cast<int>(threadIdx.x) < len) {
        my_token = tokens[threadIdx.x];
        my_u = u[threadIdx.x];
        if (my_token < 0 || my_token >= n) my_token = -1;
        if (my_token >= 0) my_x = as_float(target[static_cast<size_t>(threadIdx.x) * n + my_token]);
        if (my_token >= 0 && with_draft) my_y = as_float(draft[static_cast<size_t>(threadIdx.x) * n + my_token]);
    }
    __syncthreads();
    // a row's parts lie at r + (its first warp) to r + (its last); one lane each
    auto starts = [&](int w) { return total * w / WARPS; };
    for (int r = warp; r < n_rows; r += WARPS) {
        const long long begin = static_cast<long long>(r) * share;
        const bool has = lane < WARPS && starts(lane) < begin + share && starts(lane + 1) > begin && starts(lane) < starts(lane + 1);
        float top = has ? s.part_top[r + lane] : -INFINITY, sum = has ? s.part_sum[r + lane] : none;
        join_lanes(top, sum);
        if (lane == 0) s.top[r] = top, s.sum[r] = sum;
    }
    sync_cluster();
    for (int r = warp; r < n_rows; r += WARPS) {
        float top = -INFINITY, sum = none;
        if (lane < static_cast<int>(n_blocks)) {
            top = cluster_load(tc::in_block(tc::s32(&s.top[r]), lane));
            sum = cluster_load(tc::in_block(tc::s32(&s.sum[r]), lane));
        }
        join_lanes(top, sum);
        if (lane == 0) s.all_top[r] = top, s.all_sum[r] = sum;
    }
    __syncthreads();

    // ---- 2. the drafts
    if (static_cast<int>(threadIdx.x) < len) {
        unsigned char verdict = kRefuse;
        if (my_token >= 0) {
            const int r = static_cast<int>(threadIdx.x) * per_step;
            if (greedy) {
                verdict = my_token == __float_as_int(s.all_sum[r]) ? kAccept : kRefuse;
            } else {
                // u wq / Sq < wp / Sp; the sums are of exp((x - top) / T), the weights have a factor of their own
                const Weights wp = weights_of(s.all_top[r], temperature), wq = weights_of(s.all_top[with_draft ? r + 1 : r], temperature);
                const float other = s.all_sum[with_draft ? r + 1 : r];
                bool sure = wp.plain && wq.plain && s.all_sum[r] > 0.0f && s.all_sum[r] < INFINITY && other > 0.0f && other < INFINITY;
                double left = static_cast<double>(my_u) * static_cast<double>(s.all_sum[r]), right = weight(my_x, wp, table);
                left *= weight(wp.top, wp, table);
                if (with_draft) left *= weight(my_y, wq, table), right *= static_cast<double>(other) * weight(wq.top, wq, table);
                sure = sure && !(fabs(left - right) <= 1e-4 * fmax(fabs(left), fabs(right)));
                verdict = !sure ? kUnsure : left < right ? kAccept : kRefuse;
            }
        }
        s.verdict[threadIdx.x] = verdict;
    }
    __syncthreads();

    // ---- 3. the token behind, and what of the drafts is not sure yet
    int j = 0, next = -1;
    while (j < len && s.verdict[j] == kAccept) ++j;
    bool mine = block == 0;  // whether this block writes the answer
    if (greedy) {
        const int at = __float_as_int(s.all_sum[j]);
        next = at < n ? at : -1;
    } else {
        const double last_u = static_cast<double>(u[k]);
        Rest<T> rest;
        rest.table = table;
        rest.n = n;
        rest.inv_p = rest.inv_q = 1.0;
        auto look_at = [&] {  // row j
            rest.x = target + static_cast<size_t>(j) * n;
            rest.y = with_draft && j < len ? draft + static_cast<size_t>(j) * n : nullptr;
            rest.first = first_of(rest.x);
            rest.wp = weights_of(s.all_top[j * per_step], temperature);
            rest.wq = rest.y != nullptr ? weights_of(s.all_top[j * per_step + 1], temperature) : rest.wp;
            rest.token = j < len && !with_draft ? tokens[j] : -1;
            rest.what = rest.y != nullptr || (j < len && s.verdict[j] == kUnsure) ? Rest<T>::kSums : Rest<T>::kTarget;
        };
        look_at();
        int v0 = 0, v1 = 0, turn = 0;  // this warp's vectors
        auto deal = [&](int w) {
            const int n_vec = min((n - rest.first + VEC - 1) / VEC, from + share), size = max(0, n_vec - from);
            v0 = from + static_cast<int>(static_cast<long long>(size) * w / WARPS);
            v1 = from + static_cast<int>(static_cast<long long>(size) * (w + 1) / WARPS);
        };
        double whole = 0.0;
#pragma unroll 1
        for (;;) {
            deal(warp);
            const double2 sums = rest.sums(v0, v1);
            if (lane == 0) s.warp_sum[0][warp] = sums.x, s.warp_sum[1][warp] = sums.y;
            __syncthreads();
            if (warp == 0) {
                const double p = warp_total(lane < WARPS ? s.warp_sum[0][lane] : 0.0), q = warp_total(lane < WARPS ? s.warp_sum[1][lane] : 0.0);
                if (lane == 0) s.block_sum[turn][0] = p, s.block_sum[turn][1] = q;
            }
            sync_cluster();
            double sum_p = 0.0, sum_q = 0.0;
            if (lane < static_cast<int>(n_blocks)) {
                const uint32_t at = tc::in_block(tc::s32(&s.block_sum[turn][0]), lane);
                sum_p = cluster_load_double(at);
                sum_q = cluster_load_double(at + 8);
            }
            sum_p = warp_total(sum_p);
            sum_q = warp_total(sum_q);
            if (rest.what == Rest<T>::kSums) {
                // (the buffer of the next turn was last read before this turn's barrier)
                turn ^= 1;
                rest.inv_p = sum_p > kTiny ? 1.0 / sum_p : 0.0;
                rest.inv_q = sum_q > kTiny ? 1.0 / sum_q : 0.0;
                if (s.verdict[j] == kUnsure) {  // (only where j < len)
                    const int token = tokens[j];
                    const double p = weight(as_float(rest.x[token]), rest.wp, table) * rest.inv_p;
                    const double q = with_draft ? weight(as_float(rest.y[token]), rest.wq, table) * rest.inv_q : 1.0;
                    if (static_cast<double>(u[j]) * q < p) {
                        do ++j;
                        while (j < len && s.verdict[j] == kAccept);
                        look_at();
                        continue;
                    }
                }
                rest.what = with_draft ? Rest<T>::kRise : Rest<T>::kTarget;
                continue;
            }
            whole = sum_p;
            if (whole > kTiny || (rest.what == Rest<T>::kTarget && rest.token < 0)) break;
            turn ^= 1;
            rest.what = Rest<T>::kTarget;  // nothing is left of p: p itself
            rest.token = -1;
        }
        const double point = last_u * whole;
        if (whole > kTiny) {
            // The block, the warp's part, a part of that, the element: the first whose sums pass the point, else the last with a weight.
            double before = 0.0;
            auto pick = [&](double p) -> int {  // of the lanes' sums
                double up_to = p;
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) {
                    const double t = __shfl_up_sync(0xffffffffu, up_to, off);
                    if (lane >= off) up_to += t;
                }
                const unsigned passed = __ballot_sync(0xffffffffu, p > kTiny && before + up_to > point), some = __ballot_sync(0xffffffffu, p > kTiny);
                const int found = passed != 0 ? __ffs(static_cast<int>(passed)) - 1 : max(0, 31 - __clz(static_cast<int>(some)));
                before += __shfl_sync(0xffffffffu, up_to - p, found);
                return found;
            };
            const int chosen = pick(lane < static_cast<int>(n_blocks) ? cluster_load_double(tc::in_block(tc::s32(&s.block_sum[turn][0]), lane)) : 0.0);
            mine = static_cast<int>(block) == chosen;
            if (mine) {  // (the whole block)
                deal(pick(lane < WARPS ? s.warp_sum[0][lane] : 0.0));
                const int w0 = v0, size = v1 - v0;
                const double2 sums = rest.sums(w0 + size * warp / WARPS, w0 + size * (warp + 1) / WARPS);
                if (lane == 0) s.warp_sum[1][warp] = sums.x;
                __syncthreads();
                if (warp == 0) {
                    const int w = pick(lane < WARPS ? s.warp_sum[1][lane] : 0.0), end = w0 + size * (w + 1) / WARPS;
#pragma unroll 1
                    for (int v = w0 + size * w / WARPS; v < end; v += 32) {
                        double r[VEC], ahead = 0.0;
                        float e[VEC], d[VEC];
                        uint4 e_raw = make_uint4(0, 0, 0, 0), d_raw = e_raw;
                        const bool in = v + lane < end;
                        if (in) rest.template load<true>(v + lane, e_raw, d_raw);
                        values_of(e_raw, e);
                        values_of(d_raw, d);
#pragma unroll
                        for (int i = 0; i < VEC; ++i) r[i] = in ? rest.of(e[i], d[i], rest.first + (v + lane) * VEC + i) : 0.0, ahead += r[i];
                        double up_to = ahead;
#pragma unroll
                        for (int off = 1; off < 32; off <<= 1) {
                            const double t = __shfl_up_sync(0xffffffffu, up_to, off);
                            if (lane >= off) up_to += t;
                        }
                        double t = before + (up_to - ahead);
                        int passed = -1, some = -1;  // first weight that passes the point, last weight
#pragma unroll
                        for (int i = 0; i < VEC; ++i) {
                            t += r[i];
                            if (r[i] > 0.0) {
                                some = rest.first + (v + lane) * VEC + i;
                                if (passed < 0 && t > point) passed = some;
                            }
                        }
                        const unsigned have = __ballot_sync(0xffffffffu, passed >= 0), any = __ballot_sync(0xffffffffu, some >= 0);
                        if (have != 0) {
                            next = __shfl_sync(0xffffffffu, passed, __ffs(static_cast<int>(have)) - 1);
                            break;
                        }
                        if (any != 0) next = __shfl_sync(0xffffffffu, some, 31 - __clz(static_cast<int>(any)));
                        before += __shfl_sync(0xffffffffu, up_to, 31);
                    }
                }
            }
        }
    }
    if (mine && warp == 0) {
        for (int i = lane; i < k + 2; i += 32) out[i] = i == 0 ? j : i <= j ? tokens[i - 1] : i == j + 1 ? next : -1;
    }
    sync_cluster();  // no block's shared memory goes away under another
}

template <typename T>
struct Launcher {
    static constexpr auto kKernel = verify_kernel<T>;
    static void configure(cudaLaunchConfig_t &cfg, cudaLaunchAttribute *attr, int seqs, int blocks, cudaStream_t stream) {
        cfg.gridDim = dim3(static_cast<unsigned>(seqs) * static_cast<unsigned>(blocks));
        cfg.blockDim = dim3(kVThreads);
        cfg.stream = stream;
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = static_cast<unsigned>(blocks);
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
    }
    // clusters of so many blocks that fit on the GPU at once (cached; one device per process)
    static int fit(int blocks) {
        static int cached[kVMaxCluster + 1] = {};
        if (cached[blocks] == 0) {
            int n = 0;
            cudaLaunchConfig_t cfg{};
            cudaLaunchAttribute attr[2];
            configure(cfg, attr, 1024, blocks, nullptr);
            if ((blocks > 8 && cudaFuncSetAttribute(kKernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) ||
                cudaOccupancyMaxActiveClusters(&n, kKernel, &cfg) != cudaSuccess) {
                (void)cudaGetLastError();
                n = 0;
            }
            cached[blocks] = n > 0 ? n : -1;
        }
        return cached[blocks];
    }
    static cudaError_t launch(const VerifyArgs &a, cudaStream_t stream) {
        // As many blocks per sequence as all sequences have room for side by side, of at least 2048 elements each.  (With more, so that a second
        // round of clusters follows the first: 64 sequences of 4 drafts 180 and 249 us instead of 162.)
        int blocks = kVMaxCluster;
        while (blocks > 1 && (a.seqs > fit(blocks) || a.vocab < blocks * 2048)) --blocks;
        cudaLaunchConfig_t cfg{};
        cudaLaunchAttribute attr[2];
        configure(cfg, attr, a.seqs, blocks, stream);
        return cudaLaunchKernelEx(&cfg, kKernel, a);
    }
};

}  // namespace

cudaError_t launch_verify(const VerifyArgs &a, cudaStream_t stream) {
    return a.elem == 2 ? Launcher<__half>::launch(a, stream) : Launcher<float>::launch(a, stream);
}

}  // namespace vqm
