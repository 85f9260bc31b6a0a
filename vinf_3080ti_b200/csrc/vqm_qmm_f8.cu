// Product of e4m3 activations (a scale for each 128 columns of a row) and e4m3 weights (a scale for each block of 128 x 128) on the 5th-generation tensor
// cores:  y[t][r] = sum_b sx[b][t] sw[r / 128][b] sum_{k in block b} q[t][k] W[r][k].
//
// A stage of the ring is a block of 128 columns of both operands, by TMA.  Its products are summed by tcgen05.mma (kind::f8f6f4) into an accumulator of its own in
// tensor memory; the writers read that, and add it times the two scales to sums in registers.  So the tensor core is never read from and written to in one place: with
// two (four) accumulators the next blocks are multiplied meanwhile.
//   warp 0      one thread issues the copies
//   warp 1      one thread issues the MMAs (in the second block of a pair: passes "full" on to the first)
//   warp 2      tensor memory
//   warps 4-11  sums and outputs: two warps for each 32 lanes of tensor memory, each half of the columns
// Up to 128 activation rows: the weight rows are the lanes, the activation rows the columns (16, 32, 64 or 128).  A lane's weight scale is the block's, the activation
// scales are one for each column.
// PAIR, more than 128: two blocks of a cluster multiply 256 activation rows, which are the lanes, by 256 weight rows together (cta_group::2).  A lane then needs one factor for all
// of its 128 columns of a block; with the weight rows in the lanes it would need 128 different ones from shared memory, twice what that gives in the time of the MMAs.
// SPLIT (few tiles): the blocks (pairs) of a cluster share the columns of a tile, and exchange their sums by st.async.
//
// Every wait is bounded: on expiry the block records a status code and everybody falls through to the end.
#include <cuda.h>
#include <cuda_fp16.h>

#include "vqm_kernels.h"
#include "vqm_tiles8.cuh"

namespace vqm {
namespace {

constexpr int kRows = 128;                  // rows of a block's first operand, the lanes of tensor memory
constexpr int kABytes = kRows * kQCols;     // of a stage
constexpr int kMaxStages = 12, kMaxCluster = 8;
constexpr int kRing = 216 * 1024, kHalfRing = 106 * 1024, kPairRing = 192 * 1024, kStaging = 4096;  // (a warp's, for outputs of pairs)
constexpr int kWriters = 8, kThreads = 128 + 32 * kWriters;
// Registers of a thread: a pair's writers hold 128 sums and two sets of 32 that come from tensor memory.  The shares add up to what the block is launched with.
constexpr int kWriterRegs = 224, kOtherRegs = 56, kLaunchRegs = 168;
static_assert(128 * kOtherRegs + 32 * kWriters * kWriterRegs <= kThreads * kLaunchRegs, "registers of a block");

struct QmmF8 {
    const float *w_scales, *q_scales;
    void *y;
    unsigned *status;
    long long q_scale_pitch;
    int rows, ntok, n_k;               // n_k: blocks of 128 columns
    int row_tiles, tok_tiles;
    int stages, b_bytes;               // of the ring; bytes of a stage's second operand
    int split;                         // blocks (pairs) that share a tile's columns
    int exchange;                      // where in the ring's memory they leave sums for one another, if not where the stages are (0)
    int y_elem, add;
    int half_sm;                       // two blocks per SM
};

template <bool PAIR>
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (PAIR)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
                     : "memory");
}
// N columns of this warp's 32 lanes
template <int N>
__device__ __forceinline__ void load_sums(uint32_t at, uint32_t (&v)[N]) {
    static_assert(N == 8 || N == 16 || N == 32);
    if constexpr (N == 8)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                     : "r"(at)
                     : "memory");
    else if constexpr (N == 16)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]),
                       "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                     : "r"(at)
                     : "memory");
    else
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, "
            "%29, %30, %31}, [%32];"
            : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
              "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]),
              "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
            : "r"(at)
            : "memory");
}
__device__ __forceinline__ void loaded() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

using Two = unsigned long long;  // two fp32
__device__ __forceinline__ Two two(float x, float y) {
    Two v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
    return v;
}
__device__ __forceinline__ void add_scaled(Two &sum, uint32_t x, uint32_t y, Two scales) {
    asm("{\n\t.reg .b64 v;\n\tmov.b64 v, {%1, %2};\n\tfma.rn.f32x2 %0, v, %3, %0;\n\t}" : "+l"(sum) : "r"(x), "r"(y), "l"(scales));
}
__device__ __forceinline__ float first(Two v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float second(Two v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }

__device__ __forceinline__ float get(const float *y) { return *y; }
__device__ __forceinline__ float get(const __half *y) { return __half2float(*y); }
__device__ __forceinline__ void put(float *y, float v) { *y = v; }
__device__ __forceinline__ void put(__half *y, float v) { *y = __float2half_rn(v); }
__device__ __forceinline__ void get4(const float *y, float (&v)[4]) {
    const float4 w = *reinterpret_cast<const float4 *>(y);
    v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
}
__device__ __forceinline__ void get4(const __half *y, float (&v)[4]) {
    const uint2 w = *reinterpret_cast<const uint2 *>(y);
    const float2 p = __half22float2(*reinterpret_cast<const __half2 *>(&w.x)), q = __half22float2(*reinterpret_cast<const __half2 *>(&w.y));
    v[0] = p.x, v[1] = p.y, v[2] = q.x, v[3] = q.y;
}
__device__ __forceinline__ void put4(float *y, const float (&v)[4]) { *reinterpret_cast<float4 *>(y) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void put4(__half *y, const float (&v)[4]) {
    const __half2 p = __floats2half2_rn(v[0], v[1]), q = __floats2half2_rn(v[2], v[3]);
    *reinterpret_cast<uint2 *>(y) = make_uint2(*reinterpret_cast<const uint32_t *>(&p), *reinterpret_cast<const uint32_t *>(&q));
}
// Eight outputs `stride` apart, those of `mine` from the first `left`; reads of what they are added to go ahead of the stores.
template <typename Y>
__device__ __forceinline__ void write8(Y *y, long long stride, int left, bool add, float (&v)[8]) {
    if (add) {
        float was[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) was[j] = j < left ? get(y + j * stride) : 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += was[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (j < left) put(y + j * stride, v[j]);
}
__device__ __forceinline__ void write8_any(const QmmF8 &a, long long at, long long stride, int left, float (&v)[8]) {
    if (a.y_elem == 2) write8(static_cast<__half *>(a.y) + at, stride, left, a.add != 0, v);
    else write8(static_cast<float *>(a.y) + at, stride, left, a.add != 0, v);
}

// 32 activation rows (of the lanes) by 32 weight rows (of a lane's values), turned in shared memory so that what is written together lies together.  `room`: a
// warp's 4 KB, rows of 128 bytes whose 16-byte pieces are exchanged against bank conflicts.
template <typename Y>
__device__ __forceinline__ void write_turned(const QmmF8 &a, uint32_t room, const Two *sums, int tok0, int row0) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t to = room + lane * 128 + ((j ^ (lane & 7)) * 16);
        asm volatile("st.shared.v2.u64 [%0], {%1, %2};" ::"r"(to), "l"(sums[2 * j]), "l"(sums[2 * j + 1]) : "memory");
    }
    __syncwarp();
    Y *y = static_cast<Y *>(a.y);
    if (a.rows % 4 == 0) {  // (buffers are 16-byte aligned)
        const int piece = lane & 7, row = row0 + piece * 4;
        if (row < a.rows) {
            Y *at = y + static_cast<long long>(tok0 + (lane >> 3)) * a.rows + row;
#pragma unroll
            for (int part = 0; part < 8; part += 4) {
                float was[4][4];
                if (a.add)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (tok0 + (part + i) * 4 + (lane >> 3) < a.ntok) get4(at + (part + i) * 4ll * a.rows, was[i]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = (part + i) * 4 + (lane >> 3);
                    const uint4 w = lds128u(room + t * 128 + ((piece ^ (t & 7)) * 16));
                    float v[4] = {__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w)};
                    if (a.add)
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] += was[i][e];
                    if (tok0 + t < a.ntok) put4(at + (part + i) * 4ll * a.rows, v);
                }
            }
        }
    } else if (row0 + lane < a.rows) {
#pragma unroll 1
        for (int t = 0; t < 32 && tok0 + t < a.ntok; t += 8) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v[i]) : "r"(room + (t + i) * 128 + (((lane >> 2) ^ ((t + i) & 7)) * 16) + (lane & 3) * 4));
            write8(y + static_cast<long long>(tok0 + t) * a.rows + row0 + lane, a.rows, a.ntok - tok0 - t, a.add != 0, v);
        }
    }
}

// CW: columns of tensor memory that a writer warp reads
template <int CW, bool PAIR, bool SPLIT>
__global__ void __launch_bounds__(kThreads, !PAIR && CW <= 16 ? 2 : 1) qmm_f8_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap q_map, const QmmF8 a) {
    static_assert(!PAIR || CW == 128);
    constexpr int GROUP = PAIR ? 2 : 1, N = 2 * CW, BUFS = PAIR ? 2 : 4, TMEM = N * BUFS;
    extern __shared__ uint8_t ring_raw[];
    __shared__ __align__(8) uint64_t s_full[kMaxStages], s_empty[kMaxStages], s_acc_full[BUFS], s_acc_empty[BUFS], s_sums[kWriters];
    __shared__ __align__(16) float s_scales[PAIR ? 1 : kWriters][2][PAIR ? 4 : CW];
    __shared__ uint32_t s_tmem;
    __shared__ int s_failed, s_issued;
    const uint32_t ring = (s32(ring_raw) + 1023u) & ~1023u;  // (the swizzle works on address bits)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t in_cluster = 0;
    if constexpr (PAIR || SPLIT) asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(in_cluster));
    const int rank = PAIR ? static_cast<int>(in_cluster & 1u) : 0, part = static_cast<int>(in_cluster) / GROUP;  // place in the pair, share of the columns
    const uint32_t leader = in_cluster & ~1u;
    const int cluster = static_cast<int>(blockIdx.x) / (GROUP * a.split), n_clusters = static_cast<int>(gridDim.x) / (GROUP * a.split);
    const int k0 = SPLIT ? part * a.n_k / a.split : 0, k1 = SPLIT ? (part + 1) * a.n_k / a.split : a.n_k;
    const int n_tiles = a.row_tiles * a.tok_tiles;
    const uint32_t stage_bytes = kABytes + a.b_bytes;

    if (threadIdx.x == 0) {
        for (int s = 0; s < a.stages; ++s) {
            bar_init(s32(&s_full[s]), PAIR && rank == 0 ? 2 : 1);  // the first block of a pair hears of the second's stage
            bar_init(s32(&s_empty[s]), 1);
        }
        for (int b = 0; b < BUFS; ++b) {
            bar_init(s32(&s_acc_full[b]), 1);
            bar_init(s32(&s_acc_empty[b]), kWriters * GROUP);
        }
        for (int w = 0; w < kWriters; ++w) bar_init(s32(&s_sums[w]), 1);
        s_failed = s_issued = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(&s_tmem)), "n"(TMEM) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(&s_tmem)), "n"(TMEM) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    // Not before this block has its tensor memory: a block of the next launch, which waits for this one's end, could take all that the SM has.
    if (a.half_sm) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if constexpr (PAIR || SPLIT) cluster_sync();  // the other blocks' barriers and tensor memory exist
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = s_tmem;
    volatile int *failed = &s_failed;

    // Tiles go to clusters in turn; 8 tiles of weight rows by all tiles of activation rows follow one another, so that what is multiplied at one
    // time is a block of both that stays in L2.
    auto place = [&](int tile, int &row_tile, int &tok_tile) {
        if constexpr (!PAIR) {
            row_tile = tile, tok_tile = 0;
        } else {
            constexpr int kBand = 8;
            const int band = tile / (kBand * a.tok_tiles), first_row = band * kBand, height = min(kBand, a.row_tiles - first_row), in_band = tile - band * kBand * a.tok_tiles;
            tok_tile = in_band / height;
            row_tile = first_row + in_band - tok_tile * height;
        }
    };

    if (warp < 4) {
        if constexpr (PAIR) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == 0) {
            if (tc::elect_one()) {
                auto copy_w = [&](int stage, int k, int row_tile) {
                    copy_tile(ring + stage * stage_bytes + (PAIR ? kABytes : 0), &w_map, k * kQCols, (row_tile * GROUP + rank) * kRows, s32(&s_full[stage]));
                };
                auto copy_q = [&](int stage, int k, int tok_tile) {
                    copy_tile(ring + stage * stage_bytes + (PAIR ? 0 : kABytes), &q_map, k * kQCols, PAIR ? (tok_tile * GROUP + rank) * kRows : 0, s32(&s_full[stage]));
                };
                int issued = 0, stage = 0;
                uint32_t parity = 1;  // of the wait for a stage that is being used again
                bool ok = true;
                for (int tile = cluster; tile < n_tiles && ok; tile += n_clusters) {
                    int row_tile, tok_tile;
                    place(tile, row_tile, tok_tile);
                    int k = k0;
                    if (issued == 0) {
                        // Weights are in place before the launch (where they may not be, the caller has turned overlap off); what the kernel before this one in the
                        // stream makes, the activations, is waited for.
                        const int ahead = min(a.stages, k1 - k0);
                        for (int i = 0; i < ahead; ++i) {
                            expect(s32(&s_full[i]), stage_bytes);
                            copy_w(i, k0 + i, row_tile);
                        }
                        asm volatile("griddepcontrol.wait;" ::: "memory");
                        for (int i = 0; i < ahead; ++i) copy_q(i, k0 + i, tok_tile);
                        issued = ahead;
                        k += ahead;
                        if (ahead == a.stages) parity = 0;
                        else stage = ahead;
                    }
                    for (; k < k1; ++k) {
                        if (issued >= a.stages && !wait<false>(s32(&s_empty[stage]), parity, failed)) {
                            ok = false;
                            break;
                        }
                        expect(s32(&s_full[stage]), stage_bytes);
                        copy_w(stage, k, row_tile);
                        copy_q(stage, k, tok_tile);
                        ++issued;
                        if (++stage == a.stages) stage = 0, parity ^= 1;
                    }
                }
                s_issued = issued;
            }
            __syncwarp();
        } else if (warp == 1) {
            if (tc::elect_one()) {
                // D fp32, A and B e4m3, K-major
                const uint32_t idesc = (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(GROUP * kRows >> 4) << 24);
                int stage = 0, done = 0;
                uint32_t parity = 0;
                bool ok = true;
                for (int tile = cluster; tile < n_tiles && ok; tile += n_clusters) {
                    for (int k = k0; k < k1; ++k, ++done) {
                        const uint32_t full = s32(&s_full[stage]);
                        const int buf = done % BUFS;
                        ok = PAIR && rank == 0 ? wait<true>(full, parity, failed) : wait<false>(full, parity, failed);
                        if (!ok) break;
                        if (rank == 0) {
                            if (done >= BUFS) ok = wait<PAIR>(s32(&s_acc_empty[buf]), (done / BUFS - 1) & 1, failed);
                            if (!ok) break;
                            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                            const uint64_t a_desc = tile_desc(ring + stage * stage_bytes), b_desc = tile_desc(ring + stage * stage_bytes + kABytes);
#pragma unroll
                            for (int j = 0; j < kQCols / 32; ++j) mma_f8<PAIR>(tmem + buf * N, a_desc + 2 * j, b_desc + 2 * j, idesc, j > 0 ? 1u : 0u);
                            commit<PAIR>(s32(&s_empty[stage]), static_cast<uint32_t>(part));
                            commit<PAIR>(s32(&s_acc_full[buf]), static_cast<uint32_t>(part));
                        } else {
                            arrive_in(in_block(full, static_cast<int>(leader)));
                        }
                        if (++stage == a.stages) stage = 0, parity ^= 1;
                    }
                }
            }
            __syncwarp();
        }
        if constexpr (SPLIT) {
            if (a.exchange == 0) cluster_sync();  // (as the writers do)
            __syncwarp();
            asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        }
    } else {
        if constexpr (PAIR) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWriterRegs));
        constexpr int PART = CW < 32 ? CW : 32;  // columns of one load
        const int writer = warp - 4, lanes = warp & 3, half = writer >> 2;  // (a warp may read the 32 lanes (warp % 4) * 32 onwards)
        asm volatile("griddepcontrol.wait;" ::: "memory");
        int done = 0;
        bool ok = true;
        Two sums[CW / 2];
        int row0 = 0, tok0 = 0;  // of this lane's outputs: PAIR: activation row tok0, weight rows from row0 on; else weight row row0, activation rows from tok0 on
        for (int tile = cluster; tile < n_tiles && ok; tile += n_clusters) {
            int row_tile, tok_tile;
            place(tile, row_tile, tok_tile);
            const float *sx, *sw;
            bool has_x, has_x2 = false, has_w;
            if constexpr (PAIR) {
                tok0 = (tok_tile * GROUP + rank) * kRows + lanes * 32 + lane;
                row0 = row_tile * GROUP * kRows + half * CW;
                sx = a.q_scales + tok0, sw = a.w_scales + static_cast<size_t>(row_tile * GROUP + half) * a.n_k;
                has_x = tok0 < a.ntok, has_w = row0 < a.rows;
            } else {
                row0 = row_tile * kRows + lanes * 32 + lane;
                tok0 = half * CW;
                sx = a.q_scales + tok0 + lane, sw = a.w_scales + static_cast<size_t>(row_tile) * a.n_k;
                has_x = lane < CW && tok0 + lane < a.ntok, has_x2 = CW > 32 && tok0 + lane + 32 < a.ntok, has_w = true;
            }
#pragma unroll
            for (int j = 0; j < CW / 2; ++j) sums[j] = 0;
            // scales are on their way one block ahead
            float x_next = has_x ? sx[k0 * a.q_scale_pitch] : 0.0f, x2_next = has_x2 ? sx[k0 * a.q_scale_pitch + 32] : 0.0f, w_next = has_w ? __ldg(sw + k0) : 0.0f;
#pragma unroll 1
            for (int k = k0; k < k1; ++k, ++done) {
                const int buf = done % BUFS;
                const float x = x_next, x2 = x2_next, w = w_next;
                if (k + 1 < k1) {
                    if (has_x) x_next = sx[(k + 1) * a.q_scale_pitch];
                    if (has_x2) x2_next = sx[(k + 1) * a.q_scale_pitch + 32];
                    if (has_w) w_next = __ldg(sw + k + 1);
                }
                if constexpr (!PAIR) {
                    if (lane < CW) s_scales[writer][buf & 1][lane] = x * w;
                    if constexpr (CW > 32) s_scales[writer][buf & 1][lane + 32] = x2 * w;
                    __syncwarp();  // (and nobody reads what the next block but one replaces)
                }
                ok = warp_wait(s32(&s_acc_full[buf]), (done / BUFS) & 1, failed);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t at = tmem + buf * N + half * CW + (static_cast<uint32_t>(lanes * 32) << 16);
                uint32_t v[2][PART];
                load_sums<PART>(at, v[0]);
#pragma unroll
                for (int p = 0; p < CW / PART; ++p) {
                    loaded();
                    if (p + 1 < CW / PART) {
                        load_sums<PART>(at + (p + 1) * PART, v[(p + 1) & 1]);  // (on its way while these are added)
                    } else {
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) {
                            if constexpr (PAIR) arrive_in(in_block(s32(&s_acc_empty[buf]), static_cast<int>(leader)));
                            else bar_arrive(s32(&s_acc_empty[buf]));
                        }
                    }
                    if constexpr (PAIR) {
                        const Two s = two(x * w, x * w);
#pragma unroll
                        for (int j = 0; j < PART / 2; ++j) add_scaled(sums[p * PART / 2 + j], v[p & 1][2 * j], v[p & 1][2 * j + 1], s);
                    } else {
#pragma unroll
                        for (int j = 0; j < PART / 4; ++j) {
                            const float4 s = *reinterpret_cast<const float4 *>(&s_scales[writer][buf & 1][p * PART + 4 * j]);
                            add_scaled(sums[p * PART / 2 + 2 * j], v[p & 1][4 * j], v[p & 1][4 * j + 1], two(s.x, s.y));
                            add_scaled(sums[p * PART / 2 + 2 * j + 1], v[p & 1][4 * j + 2], v[p & 1][4 * j + 3], two(s.z, s.w));
                        }
                    }
                }
            }
            if constexpr (!SPLIT) {
                if (tile + n_clusters >= n_tiles) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
                if (!ok) break;
                if constexpr (PAIR) {
                    const uint32_t room = ring + a.stages * stage_bytes + writer * kStaging;
#pragma unroll
                    for (int p = 0; p < CW / 32; ++p) {
                        if (a.y_elem == 2) write_turned<__half>(a, room, sums + p * 16, tok0 - lane, row0 + p * 32);
                        else write_turned<float>(a, room, sums + p * 16, tok0 - lane, row0 + p * 32);
                    }
                } else if (row0 < a.rows) {
#pragma unroll
                    for (int c = 0; c < CW / 8; ++c) {
                        float v[8];
#pragma unroll
                        for (int j = 0; j < 4; ++j) v[2 * j] = first(sums[4 * c + j]), v[2 * j + 1] = second(sums[4 * c + j]);
                        write8_any(a, static_cast<long long>(tok0 + 8 * c) * a.rows + row0, a.rows, a.ntok - tok0 - 8 * c, v);
                    }
                }
            }
        }
        if constexpr (SPLIT) {
            // One tile; its sums go, 8 columns of 32 lanes at a time (a unit), to the block that writes them, and there to the same warp.
            const uint32_t room = ring + a.exchange, bar = s32(&s_sums[writer]);
            const int of_column = (kWriters + a.split - 1) / a.split;  // units of 8 columns that a block may have
            auto owner_of = [&](int c) { return (c * 9 + writer) % a.split; };
            auto room_of = [&](int c, int from, int owner) { return room + static_cast<uint32_t>((c * of_column + writer / a.split) * (a.split - 1) + (from < owner ? from : from - 1)) * 1024 + lane * 16; };
            if (a.exchange == 0) cluster_sync();  // every block's MMAs are done with its stages, where the sums go
            int mine = 0;
#pragma unroll
            for (int c = 0; c < CW / 8; ++c) {
                const int owner = owner_of(c);
                if (owner == part) {
                    ++mine;
                    continue;
                }
                // stores that count their bytes on a barrier of the block that they go to
                const uint32_t to = in_block(room_of(c, part, owner), owner * GROUP + rank), there = in_block(bar, owner * GROUP + rank);
                asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.b64 [%0], {%1, %2}, [%3];" ::"r"(to), "l"(sums[4 * c]), "l"(sums[4 * c + 1]), "r"(there) : "memory");
                asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.b64 [%0], {%1, %2}, [%3];" ::"r"(to + 512), "l"(sums[4 * c + 2]), "l"(sums[4 * c + 3]), "r"(there) : "memory");
            }
            __syncwarp();
            asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // (its other half is at the end: until then others may still send)
            asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
            if (mine > 0) {
                if (lane == 0) expect(bar, static_cast<uint32_t>(mine * (a.split - 1)) * 1024);
                const bool there = wait<true>(bar, 0, failed);  // (by every lane: it reads what others have stored)
                __syncwarp();
                if (there && ok && !*failed) {
#pragma unroll
                    for (int c = 0; c < CW / 8; ++c) {
                        if (owner_of(c) != part) continue;
                        float v[8];
#pragma unroll
                        for (int j = 0; j < 4; ++j) v[2 * j] = first(sums[4 * c + j]), v[2 * j + 1] = second(sums[4 * c + j]);
                        for (int p = 0; p < a.split; ++p) {
                            if (p == part) continue;
                            const uint32_t from = room_of(c, p, part);
                            const uint4 x = lds128u(from), z = lds128u(from + 512);
                            v[0] += __uint_as_float(x.x), v[1] += __uint_as_float(x.y), v[2] += __uint_as_float(x.z), v[3] += __uint_as_float(x.w);
                            v[4] += __uint_as_float(z.x), v[5] += __uint_as_float(z.y), v[6] += __uint_as_float(z.z), v[7] += __uint_as_float(z.w);
                        }
                        if constexpr (PAIR) {
                            if (tok0 < a.ntok) write8_any(a, static_cast<long long>(tok0) * a.rows + row0 + 8 * c, 1, a.rows - row0 - 8 * c, v);
                        } else {
                            if (row0 < a.rows) write8_any(a, static_cast<long long>(tok0 + 8 * c) * a.rows + row0, a.rows, a.ntok - tok0 - 8 * c, v);
                        }
                    }
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (s_failed && threadIdx.x == 0) {  // whichever wait gave up: the last copies land before the block may leave (this wait has a limit too)
        int left = 1 << 16;
        for (int last = max(0, s_issued - a.stages); last < s_issued; ++last)
            while (!bar_try(s32(&s_full[last % a.stages]), (last / a.stages) & 1) && --left > 0) __nanosleep(64);
    }
    __syncwarp();
    // no block's shared or tensor memory goes away under another
    if constexpr (SPLIT) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    else if constexpr (PAIR) cluster_sync();
    if (warp == 2) {
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(TMEM) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(TMEM) : "memory");
        if (lane == 0 && s_failed) atomicExch(a.status, kStatusWaitExpired);
    }
}

template <int CW, bool PAIR, bool SPLIT>
struct Variant {
    static constexpr bool kHalf = !PAIR && CW <= 16;  // two blocks per SM
    static constexpr int kGroup = PAIR ? 2 : 1, kRoom = PAIR ? kPairRing : kHalf ? kHalfRing : kRing;
    static constexpr int kSmem = kRoom + 1024 + (PAIR ? kWriters * kStaging : 0);
    static constexpr auto kKernel = qmm_f8_kernel<CW, PAIR, SPLIT>;
    static void configure(cudaLaunchConfig_t &cfg, cudaLaunchAttribute *attr, int clusters, int split, int smem, bool overlap, cudaStream_t stream) {
        cfg.gridDim = dim3(static_cast<unsigned>(clusters * split * kGroup));
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = static_cast<size_t>(smem);
        cfg.stream = stream;
        cfg.attrs = attr;
        cfg.numAttrs = launch_attributes(attr, overlap, split * kGroup);
    }
    // clusters that fit on the GPU at once, one block per SM (cached; one device per process), 0 if the kernel cannot run
    static int clusters(int split) {
        static int cached[kMaxCluster + 1] = {};
        if (cached[split] == 0) {
            int n = 0;
            cudaLaunchConfig_t cfg{};
            cudaLaunchAttribute attr[2];
            constexpr int kWhole = kRing + 1024;  // (so that there is one)
            configure(cfg, attr, 1024, split, kWhole, true, nullptr);
            cudaFuncAttributes is{};
            // (a pair's writers wait for registers that the block must have been launched with)
            if (cudaFuncGetAttributes(&is, kKernel) != cudaSuccess || (PAIR && is.numRegs < kLaunchRegs) ||
                cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem > kWhole ? kSmem : kWhole) != cudaSuccess ||
                cudaOccupancyMaxActiveClusters(&n, kKernel, &cfg) != cudaSuccess) {
                (void)cudaGetLastError();
                n = 0;
            }
            cached[split] = n > 0 ? n : -1;
        }
        return cached[split] < 0 ? 0 : cached[split];
    }
    static cudaError_t launch(const CUtensorMap &w, const CUtensorMap &q, const QmmF8 &a, bool overlap, cudaStream_t stream) {
        const int fit = clusters(a.split), tiles = a.row_tiles * a.tok_tiles;
        if (fit == 0) return cudaErrorInvalidConfiguration;
        cudaLaunchConfig_t cfg{};
        cudaLaunchAttribute attr[2];
        configure(cfg, attr, SPLIT ? tiles : (tiles < fit ? tiles : fit), a.split, kSmem, overlap, stream);
        return cudaLaunchKernelEx(&cfg, kKernel, w, q, a);
    }
};

template <int CW, bool PAIR>
cudaError_t launch(QmmF8 a, const QmmF8Args &in, cudaStream_t stream) {
    using One = Variant<CW, PAIR, false>;
    using Many = Variant<CW, PAIR, true>;
    constexpr int kStage = kABytes + (PAIR ? kRows : 2 * CW) * kQCols;
    a.tok_tiles = PAIR ? (in.ntok + 2 * kRows - 1) / (2 * kRows) : 1;
    a.row_tiles = (in.rows + One::kGroup * kRows - 1) / (One::kGroup * kRows);
    a.half_sm = One::kHalf;
    a.b_bytes = kStage - kABytes;
    // As many parts of the columns as leave every cluster room beside the others, of two blocks of columns at least.
    a.split = 1;
    const long long tiles = static_cast<long long>(a.row_tiles) * a.tok_tiles;
    if (tiles > (1ll << 30)) return cudaErrorInvalidValue;
    for (int split = 2; split <= kMaxCluster / One::kGroup && a.n_k >= 2 * split; ++split)
        if (tiles <= Many::clusters(split)) a.split = split;
    const bool brief = a.n_k <= 8 * a.split;  // a few stages for each block: what counts is how soon it begins and ends
    // Sums have memory of their own where that costs no stage or the stages are few, else they go where the stages were, one barrier of the cluster later.
    const int room = a.split > 1 ? CW / 8 * ((kWriters + a.split - 1) / a.split) * (a.split - 1) * 1024 : 0;
    a.stages = One::kRoom / kStage;
    const int beside = (One::kRoom - room) / kStage;
    if (a.split > 1 && (beside == a.stages || (brief && beside >= 3))) a.exchange = One::kRoom - room, a.stages = beside;
    if (a.stages > kMaxStages) a.stages = kMaxStages;
    CUtensorMap w, q;
    cudaError_t err = encode_rows(&w, in.w, in.cols, in.w_pitch, in.rows, kRows);
    if (err == cudaSuccess) err = encode_rows(&q, in.q, in.cols, f8_pitch(in.cols), in.ntok, PAIR ? kRows : 2 * CW);
    if (err != cudaSuccess) return err;
    return a.split > 1 ? Many::launch(w, q, a, in.overlap, stream) : One::launch(w, q, a, in.overlap, stream);
}

}  // namespace

cudaError_t launch_qmm_f8(const QmmF8Args &in, cudaStream_t stream) {
    QmmF8 a{};
    a.w_scales = in.w_scales;
    a.q_scales = in.q_scales;
    a.y = in.y;
    a.status = in.status;
    a.q_scale_pitch = f8_scale_pitch(in.ntok);
    a.rows = in.rows;
    a.ntok = in.ntok;
    a.n_k = f8_blocks(in.cols);
    a.y_elem = in.y_elem;
    a.add = in.add;
    if (in.ntok > 128) return launch<128, true>(a, in, stream);
    if (in.ntok > 64) return launch<64, false>(a, in, stream);
    if (in.ntok > 32) return launch<32, false>(a, in, stream);
    return in.ntok > 16 ? launch<16, false>(a, in, stream) : launch<8, false>(a, in, stream);
}

}  // namespace vqm
