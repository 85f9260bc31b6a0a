// Verification of drafted tokens.  Draft i of a sequence, drawn from q_i = softmax(draft logits / T), is accepted if
// u_i q_i(token) < p_i(token) with p_i = softmax(target logits / T); after the first refusal, or behind the last draft, one more token is
// drawn from max(p - q, 0) (or from p) by inverse cdf with the last random number.  That the tokens are distributed as the target's
// own holds for any q; a draft without probabilities is q = 1 at its token.
//
// One cluster per sequence, each block a slice of the vocabulary.
//   1. One pass over the logits: every row's largest and the sum of exp over it, in fp32 (exponentials by ex2, sums of one part of 16 or 32 terms after the
//      other per lane).  The blocks exchange (largest, sum) of each row through distributed shared memory.
//   2. Every block decides on all drafts.  fp32 leaves the two sides of a test uncertain by about 1e-6; where they are within a bound of that (verify_band, 1e-4 and some), and for rows
//      with values that fp32 cannot hold (infinite, undefined, too large over T), the cluster sums the row's exponentials again in 64 bits.
//   3. The token behind: which of 150000 intervals the random number falls into hangs on the 12th digit of the sums, so the one or two rows it
//      takes are summed in 64 bits: both rows' sums, then the weights by blocks and warps, then within one warp's part.
// Nothing is kept in device memory between the steps: launches on several streams and in several graphs do not meet.
//
// What bounds it: 64 sequences x 4 drafts x 151936 in fp32 take 142 us of one stream (2460 GB/s; three streams: 73.5 us a call, 4760 GB/s): 60 us are step 1, near
// the copy bandwidth, the rest the exponentials in 64 bits of two rows (eight instructions of that pipe and some twenty others each: 45 cycles per 32 of them
// and scheduler, whatever of loads, table or series is left out).  The same in fp16 114, greedy 38.5, drafts = 0 37; 75 and 149 sequences,
// a block for each and half of the SMs or two rounds, 256 and 382.  One sequence x 3 drafts: 22 to 28 us on 16 SMs, as many as a cluster takes.  Of that, half
// is the steps' latency: a vocabulary of 1000 takes 14 us.  Tried: 1024 threads, two blocks of 256 or 512 per SM (spills), a second round of
// clusters, both rows' weights kept in shared memory between their two passes (no gain).
#include <cuda_fp16.h>

#include "vqm_kernels.h"
#include "vqm_logits.cuh"
#include "vqm_tcmv.cuh"

namespace vqm {
namespace {

constexpr int kVThreads = 512, kVWarps = kVThreads / 32, kVMaxCluster = 16, kVMaxRows = 2 * 255 + 1;
constexpr int kVPart = 4;  // vectors that a lane adds up before they go to its sum
constexpr int kVTable = 128, kVCopies = 16;  // entries of 2^(j / 128), and copies: lanes that look up at random do not meet in a bank
constexpr double kVMagic = 6755399441055744.0 / kVTable;  // 1.5 * 2^52 / 128: adding it rounds to a multiple of 1 / 128
constexpr double kNoise = 1.0 / (1ull << 44);  // p - q within the rounding of the rows' sums is nothing: equal rows leave no rest
constexpr double kLn2 = 0.693147180559945309417232121458, kLog2e = 1.0 / kLn2;

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
    double warp_sum[3][kVWarps];                   // of the warps; of the row(s) being summed, of one warp's part
    double block_sum[2][2];                        // this block's, for the others; two buffers in turn
    unsigned status;
};
enum : unsigned char { kAccept, kRefuse, kUnsure };

// A row's weights exp((x - top) / T) in 64 bits, all of them times one factor near 1: 2^(x log2(e) / T - shift) with a shift that is a multiple of 1 / 128.
struct Weights {
    double scale, magic;  // log2(e) / T, kVMagic - shift
    float least;          // a smaller logit weighs 2^-1000, which counts as nothing (and so does a masked or undefined one)
    float top;
    int kind;             // of the row
};
// Rows whose logits are not taken as they are, but as 0 or -inf: only the largest count (it is infinite, or the lowest number there is), all that are not masked
// do (T above 1e30), none do.
enum : int { kOrdinary, kLargestOnly, kAllEqual, kNone };
constexpr double kTiny = 0x1p-960;

template <int N>
__device__ __forceinline__ void ordinary(const Weights &w, float *x) {
    if (w.kind == kOrdinary) return;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = (w.kind == kLargestOnly ? x[i] == w.top : w.kind == kAllEqual && x[i] > -INFINITY) ? 0.0f : -INFINITY;
}
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
        const int n = max(__double2loint(t[i]), -1000 * kVTable);  // (the logit below which nothing counts is rounded: y may be lower)
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
__device__ __forceinline__ double weight(float x, const Weights &w, const double *table) {
    double p;
    ordinary<1>(w, &x);
    powers<1>(&x, w, table, &p);
    return p > kTiny ? p : 0.0;
}
// scale, reach: log2(e) / T and 1000 over that, which a sequence's rows have in common
__device__ __forceinline__ Weights weights_of(float top, double scale, double reach) {
    constexpr float kMost = 3.402823466e38f;
    Weights w;
    w.top = top;
    w.kind = top == -INFINITY ? kNone : top == INFINITY || top <= -kMost ? kLargestOnly : scale < 1e-30 ? kAllEqual : kOrdinary;
    double at = static_cast<double>(top);
    if (w.kind != kOrdinary) {
        at = 0.0, scale = 1.0, reach = 1000.0;
    } else if (fabs(at) * scale > 4e12) {
        // the next lower number is 2^-24 of the largest away, which is 2^-200000 then: a smaller scale gives the same weights, 1 and 0
        scale = 4e12 / fabs(at);
        reach = 1000.0 / scale;
    }
    w.scale = scale;
    w.magic = kVMagic - at * scale;  // (rounds the shift)
    w.least = fmaxf(__double2float_rd(at - reach), -kMost);
    return w;
}

__device__ __forceinline__ double warp_total(double v) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}
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
    if (threadIdx.x == 0) s.status = *a.status;  // (not needed before the end: nobody waits for it there)
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
    const double scale = fmax(kLog2e / static_cast<double>(temperature), 1e-300), reach = 1000.0 * kLn2 * fmin(static_cast<double>(temperature), 1e300);
    const float c = static_cast<float>(scale);
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
            constexpr int U = kVPart;
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
                double left = static_cast<double>(my_u), right = 1.0;
                bool sure = true;
                const double band = verify_band(share / (32 * kVPart) + 2);  // (a warp has at most a block's share of a row)
#pragma unroll 1
                for (int side = 0; side < per_step; ++side) {
                    const float sum = s.all_sum[r + side];
                    const Weights w = weights_of(s.all_top[r + side], scale, reach);
                    sure = sure && w.kind == kOrdinary && sum > 0.0f && sum < INFINITY;
                    const double token_weight = weight(side ? my_y : my_x, w, table), whole = static_cast<double>(sum) * weight(w.top, w, table);
                    left *= side ? token_weight : whole;
                    right *= side ? whole : token_weight;
                }
                sure = sure && !(fabs(left - right) <= band * fmax(fabs(left), fabs(right)));
                verdict = !sure ? kUnsure : left < right ? kAccept : kRefuse;
            }
        }
        s.verdict[threadIdx.x] = verdict;
    }
    __syncthreads();

    // ---- 3. the token behind, and what of the drafts is not sure yet.  No part of this may live in local memory: a barrier of the cluster empties
    //      the L1 cache, and each access after it costs 600 cycles.  So there is one loop for all passes over the one or two rows, not a function.
    int j = 0, next = -1;
    while (j < len && s.verdict[j] == kAccept) ++j;
    bool mine = block == 0;  // whether this block writes the answer
    if (greedy) {
        const int at = __float_as_int(s.all_sum[j]);
        next = at < n ? at : -1;
    } else {
        enum { kSums, kRise, kTarget };  // passes: sums of both rows; weights max(p - q, 0); weights p
        int pass = kSums, turn = 0, skip = -1, first = 0;
        bool again = true, fine = false;  // a new row j; the last pass, over one warp's part
        const T *x = nullptr, *y = nullptr;
        Weights wp{}, wq{};
        double inv_p = 1.0, inv_q = 1.0, before = 0.0, point = 0.0;
        int v0 = 0, v1 = 0, part0 = 0, part_size = 0;
        auto above = [&](double p, double q) -> double {  // max(p - q, 0) of two weights
            const double a = __dmul_rn(p, inv_p), rise = a - __dmul_rn(q, inv_q);
            return rise > a * kNoise ? rise : 0.0;
        };
        // the first of the lanes' sums that passes the point, else the last with a weight; what is before it is added up
        auto pick = [&](double p) -> int {
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
        auto load = [&](int v, bool both, uint4 &e, uint4 &d) {
            load_vec(x, n, first, v, e);
            if (!both) return;
            if (first_of(y) == first) {
                load_vec(y, n, first, v, d);
            } else {  // the draft's row lies on another grid
                uint32_t r[4] = {};
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const int at = first + v * VEC + i;
                    const bool in = at >= 0 && at < n;
                    if constexpr (sizeof(T) == 4) r[i] = in ? __float_as_uint(as_float(y[at])) : kNothing<T>;
                    else r[i / 2] |= (in ? static_cast<uint32_t>(__half_as_ushort(y[at])) : 0xFC00u) << (16 * (i & 1));
                }
                d = make_uint4(r[0], r[1], r[2], r[3]);
            }
        };
        // weights of vector v, four at a time
        auto weights = [&](int v, bool both, const uint4 &e_raw, const uint4 &d_raw, auto use) {
            float e[VEC], d[VEC];
            values_of(e_raw, e);
            if (skip >= 0 && pass == kTarget) {
                const int at = skip - (first + v * VEC);
#pragma unroll
                for (int l = 0; l < VEC; ++l)
                    if (at == l) e[l] = -INFINITY;
            }
            ordinary<VEC>(wp, e);
            if (both) {
                values_of(d_raw, d);
                ordinary<VEC>(wq, d);
            }
#pragma unroll
            for (int i = 0; i < VEC; i += 4) {
                double p[4], q[4] = {};
                powers<4>(e + i, wp, table, p);
                if (both) powers<4>(d + i, wq, table, q);
                use(i, p, q);
            }
        };
#pragma unroll 1
        for (;;) {
            if (again) {
                x = target + static_cast<size_t>(j) * n;
                y = with_draft && j < len ? draft + static_cast<size_t>(j) * n : nullptr;
                first = first_of(x);
                wp = weights_of(s.all_top[j * per_step], scale, reach);
                wq = y != nullptr ? weights_of(s.all_top[j * per_step + 1], scale, reach) : wp;
                skip = j < len && !with_draft ? tokens[j] : -1;
                pass = y != nullptr || (j < len && s.verdict[j] == kUnsure) ? kSums : kTarget;
                const int n_vec = min((n - first + VEC - 1) / VEC, from + share);
                part0 = from, part_size = max(0, n_vec - from);
                again = false;
            }
            v0 = part0 + static_cast<int>(static_cast<long long>(part_size) * warp / WARPS);
            v1 = part0 + static_cast<int>(static_cast<long long>(part_size) * (warp + 1) / WARPS);
            const bool both = y != nullptr && pass != kTarget;
            double sum_p = 0.0, sum_q = 0.0;
            {
                uint4 e0, d0, e1, d1;
                e0 = d0 = e1 = d1 = make_uint4(0, 0, 0, 0);
                int v = v0 + lane;
                if (v < v1) load(v, both, e0, d0);
                if (v + 32 < v1) load(v + 32, both, e1, d1);
#pragma unroll 1
                for (; v < v1; v += 32) {  // (two vectors on their way)
                    const uint4 e = e0, d = d0;
                    e0 = e1, d0 = d1;
                    if (v + 64 < v1) load(v + 64, both, e1, d1);
                    weights(v, both, e, d, [&](int, const double (&p)[4], const double (&q)[4]) {
                        if (pass == kRise) {
                            sum_p += (above(p[0], q[0]) + above(p[1], q[1])) + (above(p[2], q[2]) + above(p[3], q[3]));
                        } else {
                            sum_p += (p[0] + p[1]) + (p[2] + p[3]);
                            if (both) sum_q += (q[0] + q[1]) + (q[2] + q[3]);
                        }
                    });
                }
            }
            sum_p = warp_total(sum_p);
            sum_q = warp_total(sum_q);
            if (lane == 0) s.warp_sum[fine ? 2 : 0][warp] = sum_p, s.warp_sum[1][warp] = sum_q;
            __syncthreads();
            if (fine) {
                if (warp != 0) break;
                const int w = pick(lane < WARPS ? s.warp_sum[2][lane] : 0.0), end = part0 + static_cast<int>(static_cast<long long>(part_size) * (w + 1) / WARPS);
#pragma unroll 1
                for (int v = part0 + static_cast<int>(static_cast<long long>(part_size) * w / WARPS); v < end; v += 32) {
                    double r[VEC], ahead = 0.0;
                    uint4 e = make_uint4(0, 0, 0, 0), d = e;
                    const bool in = v + lane < end;
                    if (in) load(v + lane, both, e, d);
                    weights(v + lane, both, e, d, [&](int i, const double (&p)[4], const double (&q)[4]) {
#pragma unroll
                        for (int l = 0; l < 4; ++l) {
                            const double w = pass == kRise ? above(p[l] > kTiny ? p[l] : 0.0, q[l] > kTiny ? q[l] : 0.0) : p[l] > kTiny ? p[l] : 0.0;
                            r[i + l] = in ? w : 0.0;
                            ahead += r[i + l];
                        }
                    });
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
                            some = first + (v + lane) * VEC + i;
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
                break;
            }
            if (warp == 0) {
                const double p = warp_total(lane < WARPS ? s.warp_sum[0][lane] : 0.0), q = warp_total(lane < WARPS ? s.warp_sum[1][lane] : 0.0);
                if (lane == 0) s.block_sum[turn][0] = p, s.block_sum[turn][1] = q;
            }
            sync_cluster();
            double block_p = 0.0, block_q = 0.0;
            if (lane < static_cast<int>(n_blocks)) {
                const uint32_t at = tc::in_block(tc::s32(&s.block_sum[turn][0]), lane);
                block_p = cluster_load_double(at);
                block_q = cluster_load_double(at + 8);
            }
            sum_p = warp_total(block_p);
            sum_q = warp_total(block_q);
            turn ^= 1;  // (the other buffer was last read before this turn's barrier)
            if (pass == kSums) {
                inv_p = sum_p > kTiny ? 1.0 / sum_p : 0.0;
                inv_q = sum_q > kTiny ? 1.0 / sum_q : 0.0;
                if (s.verdict[j] == kUnsure) {  // (only where j < len)
                    const int token = tokens[j];
                    const double p = weight(as_float(x[token]), wp, table) * inv_p, q = with_draft ? weight(as_float(y[token]), wq, table) * inv_q : 1.0;
                    if (static_cast<double>(u[j]) * q < p) {
                        do ++j;
                        while (j < len && s.verdict[j] == kAccept);
                        again = true;
                        continue;
                    }
                }
                pass = with_draft ? kRise : kTarget;
                continue;
            }
            if (!(sum_p > kTiny)) {
                if (pass == kTarget && skip < 0) break;  // an empty row
                pass = kTarget;                          // nothing is left of p: p itself
                skip = -1;
                continue;
            }
            point = static_cast<double>(u[k]) * sum_p;
            mine = static_cast<int>(block) == pick(block_p);
            if (!mine) break;
            // (the whole block) one warp's part again, in as many parts
            const int w = pick(lane < WARPS ? s.warp_sum[0][lane] : 0.0);
            const int begin = part0 + static_cast<int>(static_cast<long long>(part_size) * w / WARPS), end = part0 + static_cast<int>(static_cast<long long>(part_size) * (w + 1) / WARPS);
            part0 = begin, part_size = end - begin;
            fine = true;
        }
    }
    if (mine && warp == 0) {
        for (int i = lane; i < k + 2; i += 32) out[i] = s.status != 0 ? -1 : i == 0 ? j : i <= j ? tokens[i - 1] : i == j + 1 ? next : -1;
    }
    sync_cluster();  // no block's shared memory goes away under another
}

template <typename T>
struct Launcher {
    static constexpr auto kKernel = verify_kernel<T>;
    static void configure(cudaLaunchConfig_t &cfg, cudaLaunchAttribute *attr, int seqs, int blocks, bool overlap, cudaStream_t stream) {
        cfg.gridDim = dim3(static_cast<unsigned>(seqs) * static_cast<unsigned>(blocks));
        cfg.blockDim = dim3(kVThreads);
        cfg.stream = stream;
        cfg.attrs = attr;
        cfg.numAttrs = launch_attributes(attr, overlap, blocks);
    }
    // clusters of so many blocks that fit on the GPU at once (cached; one device per process)
    static int fit(int blocks) {
        static int cached[kVMaxCluster + 1] = {};
        if (cached[blocks] == 0) {
            int n = 0;
            cudaLaunchConfig_t cfg{};
            cudaLaunchAttribute attr[2];
            configure(cfg, attr, 1024, blocks, true, nullptr);
            if ((blocks > 8 && cudaFuncSetAttribute(kKernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) ||
                cudaOccupancyMaxActiveClusters(&n, kKernel, &cfg) != cudaSuccess) {
                (void)cudaGetLastError();
                n = 0;
            }
            cached[blocks] = n > 0 ? n : -1;
        }
        return cached[blocks];
    }
    static cudaError_t launch(const VerifyArgs &a, bool overlap, cudaStream_t stream) {
        // As many blocks per sequence as all sequences have room for side by side, of at least 2048 elements each.  (With more, so that a second
        // round of clusters follows the first: 64 sequences of 4 drafts 180 and 249 us instead of 162.)
        int blocks = kVMaxCluster;
        while (blocks > 1 && (a.seqs > fit(blocks) || a.vocab < blocks * 2048)) --blocks;
        cudaLaunchConfig_t cfg{};
        cudaLaunchAttribute attr[2];
        configure(cfg, attr, a.seqs, blocks, overlap, stream);
        return cudaLaunchKernelEx(&cfg, kKernel, a);
    }
};

}  // namespace

cudaError_t launch_verify(const VerifyArgs &a, bool overlap, cudaStream_t stream) {
    return a.elem == 2 ? Launcher<__half>::launch(a, overlap, stream) : Launcher<float>::launch(a, overlap, stream);
}

}  // namespace vqm
