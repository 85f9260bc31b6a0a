// Log probabilities of given tokens, the entropy of the distribution they are drawn from, and its likeliest tokens:  p = softmax(l / T),
//   out = log p(token),   entropy = - sum p log p,   the `top` largest logits, of equal ones the lowest place first.
//
// One pass over a row, in vectors of 16 bytes: each thread keeps the largest logit m it has seen, S = sum exp((l - m) / T) and U = sum exp((l - m) / T) (l - m); a new largest
// scales both.  Then  log p(t) = (l_t - m) / T - log S  and  entropy = log S - U / (S T).  The exponential of m itself, 1, is never added to the others: of a token that is all
// but certain the answers are what the others come to, log S = log(1 + (S - 1)).  So a thread keeps what came with its m (16 or 32 logits) apart from the rest of S, and the
// warp that has the row's m reads those logits again.  A row is a block's, or shared by the blocks of a cluster where there are few rows;
// sums and alternatives meet in distributed shared memory, and nothing is kept in device memory.
// The alternatives need no second pass: the `top`-th largest of the maxima of 32 groups of threads is no more than the `top`-th largest logit, because so many groups each hold
// one that is no less.  Only threads whose own largest reaches it (31 of 512 on average for 20 alternatives) hold candidates, and what they have read is read again.  Of
// n candidates each finds its own place, by counting those before it.  Rows where more tie than the list holds take a pass for each alternative.
// Rows of infinite or extreme logits, and extreme temperatures, are summed in 64 bits by one block.
//
// What bounds it.  Many rows: memory, and for fp16 the instructions as well (issue slots 51 %; the exponentials, 16 a cycle of an SM, 69 us of the 130).  2048 x 151936: fp32 189 us without
// alternatives (6.6 TB/s) and 223 with 20, fp16 113 (5.5) and 130 with one; 4 and 5 us less with the largest logit's 1 among the others.  Few rows: the steps, each of which waits
// for the one before: 1 x 151936 5.7 us, 10.2 with 20 alternatives, by one cluster of 16 blocks (more would have to meet in device memory).
#include <cuda_fp16.h>

#include "vqm_kernels.h"
#include "vqm_logits.cuh"
#include "vqm_packed.cuh"

namespace vqm {
namespace {

constexpr int kMostWarps = 16, kMaxBlocks = 16;
constexpr int kUnroll = 4;       // vectors of a thread in flight
constexpr int kList = 1024;      // candidates
constexpr int kParts = 16;       // of what a thread reads, whose largest logits are kept
constexpr float kLow = -1e30f;   // what is below counts as that in differences, so that they and their products stay finite
constexpr float kMostT = 1e20f, kLeastT = 1e-30f;  // temperatures that fp32 works with: a masked logit, at -1e30 or less, still comes to nothing

using Key = unsigned long long;
// A logit and its place as one number, larger for what comes first: by value, then by the lower place.  0: nothing (masked).
__device__ __forceinline__ Key key_of(float v, int i) {
    if (!(v > -INFINITY)) return 0;
    const uint32_t b = __float_as_uint(v == 0.0f ? 0.0f : v);  // (the zeros are equal)
    return static_cast<Key>((b & 0x80000000u) != 0 ? ~b : b | 0x80000000u) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(i));
}
__device__ __forceinline__ int place_of(Key key) { return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(key)); }
__device__ __forceinline__ float value_of(Key key) {
    const uint32_t b = static_cast<uint32_t>(key >> 32);
    return __uint_as_float((b & 0x80000000u) != 0 ? b & 0x7FFFFFFFu : ~b);
}
__device__ __forceinline__ float undefined() { return __uint_as_float(0x7FFFFFFFu); }

// The largest of some vectors (NaN counts as nothing).
__device__ __forceinline__ float largest(const uint4 (&w)[kUnroll], const float *) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
        m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(w[i].x), __uint_as_float(w[i].y)), fmaxf(__uint_as_float(w[i].z), __uint_as_float(w[i].w))));
    return m;
}
__device__ __forceinline__ float largest(const uint4 (&w)[kUnroll], const __half *) {
    auto half2_of = [](uint32_t v) { return *reinterpret_cast<const __half2 *>(&v); };
    __half2 m = half2_of(0xFC00FC00u);
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) m = __hmax2(m, __hmax2(__hmax2(half2_of(w[i].x), half2_of(w[i].y)), __hmax2(half2_of(w[i].z), half2_of(w[i].w))));
    return fmaxf(__low2float(m), __high2float(m));
}

struct Sums {
    float m, u;       // the largest so far (kLow: none), and U
    float s, with_m;  // S in two parts, the second from the vectors that brought m: those hold a 1, next to which small terms lose their digits
};
template <typename T, int THREADS>
__device__ __forceinline__ float add_vectors(Sums &a, const uint4 (&w)[kUnroll], int at, float c, int *brought) {  // returns their largest
    const float most = largest(w, static_cast<const T *>(nullptr));
    const bool more = most > a.m;
    if (more) {
        const float d = a.m - most, f = ex2(d * c), s = a.s + a.with_m;
        a.u = f * fmaf(d, s, a.u);
        a.s = f * s;
        a.m = most;
        brought[threadIdx.x] = at;
    }
    const Two minus = two(-a.m, -a.m), cc = two(c, c);
    Two s = 0, u = 0;
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
        float x[kVec<T>];
        values_of(w[i], x);
#pragma unroll
        for (int e = 0; e < kVec<T>; e += 2) {
            float d0, d1, t0, t1;
            both(add2(two(x[e], x[e + 1]), minus), d0, d1);
            const Two d = two(fmaxf(d0, kLow), fmaxf(d1, kLow));
            both(mul2(d, cc), t0, t1);
            const Two p = two(ex2(t0), ex2(t1));
            s = add2(s, p);
            u = fma2(p, d, u);
        }
    }
    float s0, s1, u0, u1;
    both(s, s0, s1);
    both(u, u0, u1);
    const float here = s0 + s1;
    if (more) a.with_m = here;
    else a.s += here;
    a.u += u0 + u1;
    return most;
}

template <int THREADS>
struct Shared {
    float most[THREADS / 32][32];   // largest logits of the threads
    float part[2][kMostWarps];
    int ones[kMostWarps];           // exponentials that are 1
    alignas(16) Key list[kList];    // candidates
    union {
        struct {
            alignas(16) float groups[THREADS / 32][32];  // the warps' copies of the groups' largest
            int brought[THREADS];                        // the first of the vectors that each thread's largest logit came with
        };
        Key theirs[THREADS == 512 ? kMaxBlocks : 1][kMaxTop];  // later on: the alternatives of a cluster's blocks
    };
    Key best[kMaxTop];              // this block's, in order
    Key key[kMostWarps];
    double wide[kMostWarps];
    float sums[4];                  // this block's m, S but for what is 1, U, and how many are 1
    int count;
    unsigned status;
};

__device__ __forceinline__ float warp_largest(float v) {
    float m;
    asm volatile("redux.sync.max.f32 %0, %1, 0xFFFFFFFF;" : "=f"(m) : "f"(v));
    return m;
}
template <int THREADS, typename V, typename F>
__device__ V over_block(V v, V (&room)[kMostWarps], F &&join) {
    for (int off = 16; off > 0; off >>= 1) v = join(v, __shfl_xor_sync(0xFFFFFFFFu, v, off));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) room[threadIdx.x >> 5] = v;
    __syncthreads();
    v = room[0];
    for (int w = 1; w < THREADS / 32; ++w) v = join(v, room[w]);
    return v;
}
// The first `want` of s.list[0, n) in order, by the whole block, to s.best; zeros behind the last.  s.list has room for zeros up to a multiple of 4.
template <int THREADS>
__device__ __forceinline__ void rank_list(Shared<THREADS> &s, int n, int want) {
    if (threadIdx.x < kMaxTop) s.best[threadIdx.x] = 0;
    if (threadIdx.x < 4 && n % 4 != 0 && threadIdx.x >= static_cast<unsigned>(n % 4)) s.list[n / 4 * 4 + threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += THREADS) {
        const Key mine = s.list[i];
        int before = 0;
        for (int j = 0; j < n; j += 4) {
            const ulonglong2 p = *reinterpret_cast<const ulonglong2 *>(s.list + j), q = *reinterpret_cast<const ulonglong2 *>(s.list + j + 2);
            before += (p.x > mine) + (p.y > mine) + (q.x > mine) + (q.y > mine);
        }
        if (mine != 0 && before < want) s.best[before] = mine;
    }
    __syncthreads();
}
// The same of all of a slice [begin, end), a pass for each.
template <typename T, int THREADS>
static __device__ __noinline__ void rank_by_passes(Shared<THREADS> &s, const T *x, int begin, int end, int want) {
    Key last = ~0ull;
    for (int k = 0; k < want; ++k) {
        Key most = 0;
        if (last != 0)
            for (int i = begin + static_cast<int>(threadIdx.x); i < end; i += THREADS) {
                const Key key = key_of(as_float(x[i]), i);
                if (key < last && key > most) most = key;
            }
        last = over_block<THREADS>(most, s.key, [](Key p, Key q) { return p > q ? p : q; });
        if (threadIdx.x == 0) s.best[k] = last;
    }
    __syncthreads();
}
// log S and the entropy in 64 bits, by the whole block.
template <typename T, int THREADS>
static __device__ __noinline__ void wide_sums(Shared<THREADS> &s, const T *x, int n, float top, double inverse, bool flat, double &log_sum, double &entropy) {
    double sum = 0.0, weighted = 0.0, ones = 0.0;
    for (int i = threadIdx.x; i < n; i += THREADS) {
        const float v = as_float(x[i]);
        if (!(v > -INFINITY)) continue;
        if (v == top || flat) {
            ones += 1.0;
            continue;
        }
        const double d = top == INFINITY ? -INFINITY : (static_cast<double>(v) - static_cast<double>(top)) * inverse, e = exp(d);
        sum += e;
        if (e > 0.0) weighted -= e * d;
    }
    auto plus = [](double p, double q) { return p + q; };
    sum = over_block<THREADS>(sum, s.wide, plus);
    weighted = over_block<THREADS>(weighted, s.wide, plus);
    ones = over_block<THREADS>(ones, s.wide, plus);
    const double rest = ones - 1.0 + sum;
    log_sum = ones > 0.0 ? log1p(rest) : 0.0;
    entropy = ones > 0.0 ? log_sum + weighted / (1.0 + rest) : 0.0;
}

__device__ __forceinline__ uint32_t in_cluster(const void *p, int block) {
    uint32_t at;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(block));
    return at;
}
__device__ __forceinline__ float load_float(uint32_t at) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ Key load_key(uint32_t at) {
    Key v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void sync_cluster() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <typename T, int THREADS, int PER_SM>
__global__ void __launch_bounds__(THREADS, PER_SM) logprobs_kernel(const LogprobsArgs a, const int n_blocks) {
    __shared__ Shared<THREADS> s;
    __shared__ float part_room[kParts * THREADS];
    constexpr int VEC = kVec<T>, WARPS = THREADS / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = a.vocab;
    const int row = static_cast<int>(blockIdx.x) / n_blocks, block = static_cast<int>(blockIdx.x) % n_blocks;
    const T *x = static_cast<const T *>(a.logits) + static_cast<size_t>(row) * n;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const float given = a.temperature != nullptr ? a.temperature[row] : 1.0f;
    const bool greedy = !(given > 0.0f);
    const bool ordinary = given >= kLeastT && given <= kMostT;  // of the temperature
    const float c = ordinary ? 1.4426950408889634f / given : 1.0f;
    if (threadIdx.x == 0) {
        s.count = 0;
        s.status = *a.status;
    }

    // What the answer needs besides is read ahead of the row, where rows are few (1 x 151936 5.3 and 5.0 us); the registers cost many rows more than that (108.6 and 109.8).
    constexpr bool kAhead = THREADS == 512;
    auto token_at = [&](int &token, float &v) {
        token = a.tokens[row];
        v = token >= 0 && token < n ? as_float(x[token]) : -INFINITY;
    };
    int token = -1;
    float asked = -INFINITY;
    if (kAhead && threadIdx.x == 32 && block == 0) token_at(token, asked);

    // this block's vectors
    const int first = first_of(x);  // index of vector 0's first element
    const int vectors = (n - first + VEC - 1) / VEC;
    const int begin = static_cast<int>(static_cast<long long>(vectors) * block / n_blocks), end = static_cast<int>(static_cast<long long>(vectors) * (block + 1) / n_blocks);
    const uint4 *const vector0 = reinterpret_cast<const uint4 *>(x + first);
    const int whole = min(end, vectors - 1);  // vectors before it (but for the row's first) hold nothing else
    const int per_part = (end - begin + kParts * kUnroll * THREADS - 1) / (kParts * kUnroll * THREADS);  // turns of the loop
    const int want = a.top > 0 ? a.top : greedy ? 1 : 0;
    float(*const part_most)[THREADS] = reinterpret_cast<float(*)[THREADS]>(part_room);
    Sums sums{kLow, 0.0f, 0.0f, 0.0f};
    float in_part = -INFINITY;
    int part = 0, turn = 0;
#pragma unroll 1
    for (int v = begin + static_cast<int>(threadIdx.x); v < end; v += kUnroll * THREADS) {
        uint4 w[kUnroll];
        if (v > 0 && v + (kUnroll - 1) * THREADS < whole) {
#pragma unroll
            for (int i = 0; i < kUnroll; ++i) w[i] = vector0[v + i * THREADS];
        } else {
#pragma unroll
            for (int i = 0; i < kUnroll; ++i) {
                if (v + i * THREADS < end) load_vec(x, n, first, v + i * THREADS, w[i]);
                else w[i] = make_uint4(kNothing<T>, kNothing<T>, kNothing<T>, kNothing<T>);
            }
        }
        in_part = fmaxf(in_part, add_vectors<T, THREADS>(sums, w, v, c, s.brought));
        if (want > 0 && ++turn == per_part) {
            part_most[part++][threadIdx.x] = in_part;
            in_part = -INFINITY;
            turn = 0;
        }
    }
    if (turn > 0) part_most[part++][threadIdx.x] = in_part;

    // the largest of each group, the threads of one place in their warps, and the block's
    s.most[warp][lane] = sums.m;
    __syncthreads();
    float mine = s.most[0][lane];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) mine = fmaxf(mine, s.most[w][lane]);
    const float all = warp_largest(mine);
    // The largest logit's 1 is counted, not added; its thread's warp adds up again what it came with.  (Of several such threads one in each warp: with two ones nothing is certain.)
    const int owner = __ffs(__ballot_sync(0xFFFFFFFFu, sums.m == all && all > kLow)) - 1;
    const float f = ex2((sums.m - all) * c), held = sums.s + sums.with_m;
    float sum = lane == owner ? sums.s : held * f, weighted = f * fmaf(sums.m - all, held, sums.u);
    int ones = 0;
    if (owner >= 0 && lane < kUnroll * VEC) {
        const int vector = s.brought[warp * 32 + owner] + lane / VEC * THREADS, i = first + vector * VEC + lane % VEC;
        const float v = vector < end && i >= 0 && i < n ? as_float(x[i]) : -INFINITY;
        if (v == all) ones = 1;
        else sum += ex2(fmaxf(v - all, kLow) * c);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
        weighted += __shfl_xor_sync(0xFFFFFFFFu, weighted, off);
    }
    ones = __reduce_add_sync(0xFFFFFFFFu, ones);
    if (lane == 0) s.part[0][warp] = sum, s.part[1][warp] = weighted, s.ones[warp] = ones;

    if (want > 0) {
        // The want-th largest group: the largest value that so many reach.  Where that is out of what the sums tell apart, all logits are candidates.
        float least = all;
        if (want > 1) {
            float *const group = s.groups[warp];
            group[lane] = mine;
            __syncwarp();
            int reach = 0;
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
                const float4 g = *reinterpret_cast<const float4 *>(group + j);
                reach += (g.x >= mine) + (g.y >= mine) + (g.z >= mine) + (g.w >= mine);
            }
            least = warp_largest(reach >= want ? mine : -INFINITY);
        }
        const bool any = !(least > kLow);
        if (any) least = -INFINITY;
        auto offer = [&](const uint4 &w, int v) {
            float value[VEC];
            values_of(w, value);
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (value[e] >= least && value[e] > -INFINITY) {
                    const int at = atomicAdd(&s.count, 1);
                    if (at < kList) s.list[at] = key_of(value[e], first + v * VEC + e);
                }
        };
        if (any) {
            for (int v = begin + static_cast<int>(threadIdx.x); v < end && s.count <= kList; v += THREADS) {  // (a count beyond the list's size is all that is asked then)
                uint4 w;
                load_vec(x, n, first, v, w);
                offer(w, v);
            }
        } else {
            // a thread reads those parts again that hold one
            unsigned parts = 0;
            if (sums.m >= least)
                for (int p = 0; p < part; ++p) parts |= part_most[p][threadIdx.x] >= least ? 1u << p : 0u;
            for (; parts != 0; parts &= parts - 1) {
                const int from = begin + static_cast<int>(threadIdx.x) + (__ffs(parts) - 1) * per_part * kUnroll * THREADS;
                for (int t = 0; t < per_part; ++t) {
                    uint4 w[kUnroll];
#pragma unroll
                    for (int i = 0; i < kUnroll; ++i) {
                        const int v = from + (t * kUnroll + i) * THREADS;
                        if (v < end) load_vec(x, n, first, v, w[i]);
                        else w[i] = make_uint4(kNothing<T>, kNothing<T>, kNothing<T>, kNothing<T>);
                    }
#pragma unroll
                    for (int i = 0; i < kUnroll; ++i) offer(w[i], from + (t * kUnroll + i) * THREADS);
                }
            }
        }
        __syncthreads();
        const int found = s.count;
        if (found <= kList) rank_list<THREADS>(s, found, want);
        else rank_by_passes<T, THREADS>(s, x, max(0, first + begin * VEC), min(n, first + end * VEC), want);
    } else {
        __syncthreads();
    }
    if (warp == 0) {
        float p = lane < WARPS ? s.part[0][lane] : 0.0f, q = lane < WARPS ? s.part[1][lane] : 0.0f;
        const int o = __reduce_add_sync(0xFFFFFFFFu, lane < WARPS ? s.ones[lane] : 0);
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) {
            p += __shfl_xor_sync(0xFFFFFFFFu, p, off);
            q += __shfl_xor_sync(0xFFFFFFFFu, q, off);
        }
        if (lane == 0) s.sums[0] = all, s.sums[1] = p, s.sums[2] = q, s.sums[3] = static_cast<float>(o);
    }
    if (n_blocks > 1) {
        sync_cluster();
        if (block != 0) {
            sync_cluster();  // (until then the first block reads what is here)
            return;
        }
    } else {
        __syncthreads();
    }

    // The first block joins the others' sums (every warp for itself) and alternatives.
    float top = kLow;
    double rest = 0.0, product = 0.0;  // S - 1, U
    {
        float m = kLow, p = 0.0f, q = 0.0f, o = 0.0f;
        if (lane < n_blocks) {
            const uint32_t at = in_cluster(s.sums, lane);
            m = load_float(at), p = load_float(at + 4), q = load_float(at + 8), o = load_float(at + 12);
        }
        top = m;
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, off));
        const float g = ex2((m - top) * c);
        product = static_cast<double>(g * fmaf(m - top, p + o, q));
        rest = m == top ? static_cast<double>(p) : static_cast<double>((p + o) * g);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
            rest += __shfl_xor_sync(0xFFFFFFFFu, rest, off);
            product += __shfl_xor_sync(0xFFFFFFFFu, product, off);
        }
        rest += static_cast<double>(static_cast<int>(__reduce_add_sync(0xFFFFFFFFu, m == top ? static_cast<int>(o) : 0)) - 1);
    }
    if (want > 0 && n_blocks > 1) {
        // Of lists in order, if r of them have a q-th key no less than some key, and r q is `want` at least, what is under that key is not asked for.
        for (int i = threadIdx.x; i < n_blocks * want; i += THREADS) s.theirs[i / want][i % want] = load_key(in_cluster(s.best, i / want) + static_cast<uint32_t>(i % want) * 8);
        if (threadIdx.x == 0) s.count = 0;
        __syncthreads();
        const int q = warp + 1, r = (want + q - 1) / q;
        Key least = 0;
        if (q <= want && r <= n_blocks) {
            const Key key = lane < n_blocks ? s.theirs[lane][q - 1] : 0;
            int before = 0;
#pragma unroll
            for (int j = 0; j < kMaxBlocks; ++j) {
                const Key other = __shfl_sync(0xFFFFFFFFu, key, j);
                before += other > key || (other == key && j < lane);
            }
            least = __shfl_sync(0xFFFFFFFFu, key, __ffs(__ballot_sync(0xFFFFFFFFu, before == r - 1)) - 1);
        }
        if (lane == 0) s.key[warp] = least;
        __syncthreads();
        for (int w = 0; w < WARPS; ++w) least = s.key[w] > least ? s.key[w] : least;
        for (int i = threadIdx.x; i < n_blocks * want; i += THREADS) {
            const Key key = s.theirs[i / want][i % want];
            if (key != 0 && key >= least) s.list[atomicAdd(&s.count, 1)] = key;
        }
        __syncthreads();
        rank_list<THREADS>(s, s.count, want);
    }
    if (n_blocks > 1) sync_cluster();  // nothing of the others is read any more

    const bool in_reach = top > kLow && top < -kLow;
    if (warp > 1 && (greedy || (in_reach && ordinary))) return;
    double log_sum = 0.0, entropy = 0.0, inverse = 1.0 / static_cast<double>(given);
    const bool flat = given > 1e30f;
    bool none = false;
    if (greedy) {
        none = s.best[0] == 0;
    } else if (in_reach && ordinary) {
        log_sum = log1p(rest);
        entropy = log_sum - product / ((1.0 + rest) * static_cast<double>(given));
    } else {
        if (!in_reach) {  // the largest as it is
            float m = -INFINITY;
            for (int i = threadIdx.x; i < n; i += THREADS) m = fmaxf(m, as_float(x[i]));
            top = over_block<THREADS>(m, s.part[0], [](float p, float q) { return fmaxf(p, q); });
        }
        none = top == -INFINITY;
        wide_sums<T, THREADS>(s, x, n, top, inverse, flat && top < INFINITY, log_sum, entropy);
    }
    auto answer = [&](float v, int place) -> float {
        if (s.status != 0) return undefined();
        if (none || !(v > -INFINITY)) return -INFINITY;
        if (greedy) return place == place_of(s.best[0]) ? 0.0f : -INFINITY;
        if (v == top || (flat && top < INFINITY)) return static_cast<float>(-log_sum);
        return top == INFINITY ? -INFINITY : static_cast<float>((static_cast<double>(v) - static_cast<double>(top)) * inverse - log_sum);
    };
    if (threadIdx.x == 32) {
        if (!kAhead) token_at(token, asked);
        a.out[row] = answer(asked, token);
        if (a.entropy != nullptr) a.entropy[row] = s.status != 0 ? undefined() : none || greedy ? 0.0f : static_cast<float>(entropy > 0.0 ? entropy : 0.0);
    }
    if (threadIdx.x < static_cast<unsigned>(a.top)) {
        const Key key = s.best[threadIdx.x];
        const size_t to = static_cast<size_t>(row) * a.top + threadIdx.x;
        a.top_ids[to] = key != 0 && s.status == 0 ? place_of(key) : -1;
        if (a.top_out != nullptr) a.top_out[to] = answer(key != 0 ? value_of(key) : -INFINITY, place_of(key));
    }
}

// A block of 256 threads for each row; where there are few rows, the blocks of a cluster, of 512.
template <typename T, bool SHARED>
struct Launcher {
    static constexpr int kThreads = SHARED ? 512 : 256;
    static constexpr auto kKernel = logprobs_kernel<T, kThreads, SHARED ? 2 : 5>;
    static void configure(cudaLaunchConfig_t &cfg, cudaLaunchAttribute *attr, int rows, int blocks, bool overlap, cudaStream_t stream) {
        cfg.gridDim = dim3(static_cast<unsigned>(rows) * static_cast<unsigned>(blocks));
        cfg.blockDim = dim3(kThreads);
        cfg.stream = stream;
        cfg.attrs = attr;
        cfg.numAttrs = launch_attributes(attr, overlap, SHARED ? blocks : 0);
    }
    // clusters of so many blocks that fit on the GPU at once (cached; one device per process)
    static int fit(int blocks) {
        static int cached[kMaxBlocks + 1] = {};
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
    static cudaError_t launch(const LogprobsArgs &a, int blocks, bool overlap, cudaStream_t stream) {
        cudaLaunchConfig_t cfg{};
        cudaLaunchAttribute attr[2];
        configure(cfg, attr, a.rows, blocks, overlap, stream);
        return cudaLaunchKernelEx(&cfg, kKernel, a, blocks);
    }
};
template <typename T>
cudaError_t launch(const LogprobsArgs &a, bool overlap, cudaStream_t stream) {
    // As many blocks of 512 threads per row as all rows have room for side by side, of at least 4096 elements each.  With more rows, or short ones, what counts is how many
    // rows at different steps an SM holds: five blocks of 256 threads.  (151936, fp32, 20 alternatives: 149 rows 30 us and 48, 300 rows 59 and 56; 300 rows of 5000 11 and 7.)
    for (int blocks = kMaxBlocks; blocks > 0; blocks /= 2)
        if (a.vocab >= (blocks > 1 ? blocks : 2) * 4096 && a.rows <= Launcher<T, true>::fit(blocks)) return Launcher<T, true>::launch(a, blocks, overlap, stream);
    return Launcher<T, false>::launch(a, 1, overlap, stream);
}

}  // namespace

cudaError_t launch_logprobs(const LogprobsArgs &a, bool overlap, cudaStream_t stream) {
    return a.elem == 2 ? launch<__half>(a, overlap, stream) : launch<float>(a, overlap, stream);
}

}  // namespace vqm
