// Product of 8-bit integers on the 5th-generation tensor cores:  y[t][r] = sx[t] sw[r] sum_k q[t][k] W[r][k],  sums in 32-bit integers, exact.
//
// The weight rows are the rows of the accumulator (lanes of tensor memory), the activation rows its columns: an output row of 32 lanes is
// then 128 consecutive bytes, and a lane needs one weight scale.  Both operands come by TMA in 128-byte swizzled tiles of 128 columns, go
// through a ring of stages, and are multiplied by tcgen05.mma (kind::i8).
//   warp 0      one thread issues the copies
//   warp 1      one thread issues the MMAs (in the second block of a pair: passes "full" on to the first)
//   warp 2      tensor memory
//   warps 4-11  outputs: two warps for each 32 lanes
// PAIR (more than 256 activation rows): two blocks of a cluster multiply 256 weight rows by up to 256 activation rows together (cta_group::2), each holding
// half of both; they take tile after tile, and the outputs of one are written while the next is multiplied (two accumulators).
// SPLIT (few tiles): the blocks (pairs) of a cluster share the columns of a tile; sums are integers, so how they are split does not show in the result.
// Every output is the same whatever else is in its launch.
//
// What bounds it.  Few rows: memory, and 3 us of start and end (17408 x 5120 with 1 row: 16.6 us of one stream, 5390 GB/s; 151936 x 5120 with 4: 124 us, 6300).
// Many: the MMAs, 512 cycles a stage of a pair, at 73 % of their rate for 2048 rows, 56 % for 512 (two rounds of tiles, start and end), and the power cap:
// 17408 x 5120 x 4096 takes 225 us (3240 TOP/s) in a burst and 265 at the 1530 MHz that 1000 W leave.  1024 x 5120 with 4 rows: 6.6 us, of which 2 are
// the exchange of sums.  What it took: the loop that issues the MMAs in one thread, with waits that look at their barrier only (4096 rows: 307 and 299
// us); outputs loaded 16 columns ahead, scales in shared memory, no choice of types inside (a tile's outputs took 10 us, as long as its MMAs: 299 and
// 262); two blocks per SM for few rows (5120 x 17408 with 24: 15.6 and 13.9).  Tried: weights fetched into L2 8 or 24 stages ahead of their copies, 16.6
// and 19.7 or 22.0 us for one row.  In between, 17408 x 5120 of one stream: 33 rows 18.0 us, 64 18.4, 128 19.6, 256 25.4: a block's one tile is written
// after its products.  Products onto what is there read an output behind the one before: 4 rows 18.7, 256 rows 81.
//
// Every wait is bounded: on expiry the block records a status code and everybody falls through to the end.
#include <cuda.h>
#include <cuda_fp16.h>

#include "vqm_kernels.h"
#include "vqm_tiles8.cuh"

namespace vqm {
namespace {

constexpr int kQRows = 128;                         // weight rows of a block's tile
constexpr int kQA = kQRows * kQCols;                // bytes of a stage's weights
constexpr int kQMaxN = 256, kQMaxStages = 12, kQMaxSplit = 8;
// Shared memory of the stages.  Blocks of few activation rows, which wait for memory, take half an SM: those of the next launch are there already, with
// their first weights on the way, while the last outputs are written.
constexpr int kQRing = 216 * 1024, kQHalfRing = 108 * 1024;
constexpr int kQWriters = 8, kQThreads = 128 + 32 * kQWriters;

struct QmmTc {
    const float *w_scales, *q_scales;
    void *y;
    unsigned *status;
    int rows, ntok, n_k;               // n_k: stages of a whole row
    int n, row_tiles, tok_tiles;       // activation rows of a tile, a multiple of 16 (pairs: 32)
    int stages, b_bytes;               // of the ring; bytes of a block's activations in a stage
    int acc_cols, tmem_cols;           // tensor-memory columns from one accumulator to the next, and in all
    int split;                         // blocks (pairs) that share a tile's columns
    int exchange;                      // where in the ring's memory they leave sums for one another, if not where the stages are (0)
    int y_elem, add;
    int half_sm;                       // two blocks per SM
};

// A wait by one lane for its warp.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int *failed) {
    int ok = 1;
    if ((threadIdx.x & 31) == 0) ok = wait<false>(bar, parity, failed) ? 1 : 0;
    __syncwarp();
    return __shfl_sync(0xFFFFFFFFu, ok, 0) != 0;
}
__device__ __forceinline__ void arrive_in(uint32_t cluster_addr) { asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory"); }
template <bool PAIR>
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (PAIR)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
                     : "memory");
}
template <int N>
__device__ __forceinline__ void load_sums(uint32_t at, int (&v)[N]) {
    __syncwarp();
    if constexpr (N == 8)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                     : "r"(at)
                     : "memory");
    else
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]),
                       "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                     : "r"(at)
                     : "memory");
}
__device__ __forceinline__ void loaded() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void put(float *y, float v, bool add) { *y = add ? *y + v : v; }
__device__ __forceinline__ void put(__half *y, float v, bool add) { *y = __float2half_rn(add ? __half2float(*y) + v : v); }

// Outputs of this lane's weight row for N activation rows from `tok` on, whose scales are in shared memory.
template <typename Y, bool ADD, int N>
__device__ __forceinline__ void write_rows(const QmmTc &a, const int (&v)[N], int row, int tok, float w_scale, const float *scales) {
    const int left = a.ntok - tok;
    Y *y = static_cast<Y *>(a.y) + static_cast<size_t>(tok) * a.rows + row;
    const bool mine = row < a.rows;
#pragma unroll
    for (int j = 0; j < N; ++j, y += a.rows) {
        const float out = static_cast<float>(v[j]) * scales[j] * w_scale;
        if (mine && j < left) put(y, out, ADD);
    }
}
template <int N>
__device__ __forceinline__ void write_any(const QmmTc &a, const int (&v)[N], int row, int tok, float w_scale, const float *scales) {
    if (a.y_elem == 2) a.add ? write_rows<__half, true>(a, v, row, tok, w_scale, scales) : write_rows<__half, false>(a, v, row, tok, w_scale, scales);
    else a.add ? write_rows<float, true>(a, v, row, tok, w_scale, scales) : write_rows<float, false>(a, v, row, tok, w_scale, scales);
}
// A tile's activation scales, by the writers (256 threads), and a barrier among them.
__device__ __forceinline__ void fetch_scales(const QmmTc &a, int tok, float *to) {
    const int i = static_cast<int>(threadIdx.x) - 128;
    if (i < a.n) to[i] = tok + i < a.ntok ? a.q_scales[tok + i] : 0.0f;
    asm volatile("bar.sync 1, %0;" ::"n"(32 * kQWriters) : "memory");
}

template <bool PAIR, bool SPLIT>
__global__ void __launch_bounds__(kQThreads, PAIR ? 1 : 2) qmm_i8_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap q_map, const QmmTc a) {
    constexpr int GROUP = PAIR ? 2 : 1;
    extern __shared__ uint8_t ring_raw[];
    __shared__ __align__(8) uint64_t s_full[kQMaxStages], s_empty[kQMaxStages], s_acc_full[2], s_acc_empty[2];
    __shared__ __align__(8) uint64_t s_sums;
    __shared__ float s_scales[2][kQMaxN];
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
    const uint32_t stage_bytes = kQA + a.b_bytes;

    if (threadIdx.x == 0) {
        for (int s = 0; s < a.stages; ++s) {
            bar_init(s32(&s_full[s]), PAIR && rank == 0 ? 2 : 1);  // the first block of a pair hears of the second's stage
            bar_init(s32(&s_empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            bar_init(s32(&s_acc_full[b]), 1);
            bar_init(s32(&s_acc_empty[b]), kQWriters * GROUP);
        }
        bar_init(s32(&s_sums), 1);
        s_failed = s_issued = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(&s_tmem)), "r"(a.tmem_cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(&s_tmem)), "r"(a.tmem_cols) : "memory");
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
        constexpr int kBand = 8;
        const int band = tile / (kBand * a.tok_tiles), first = band * kBand, height = min(kBand, a.row_tiles - first), in_band = tile - band * kBand * a.tok_tiles;
        tok_tile = in_band / height;
        row_tile = first + in_band - tok_tile * height;
    };

    if (warp == 0) {
        if (tc::elect_one()) {
            auto copy_w = [&](int stage, int k, int row_tile) { copy_tile(ring + stage * stage_bytes, &w_map, k * kQCols, (row_tile * GROUP + rank) * kQRows, s32(&s_full[stage])); };
            auto copy_q = [&](int stage, int k, int tok_tile) {
                copy_tile(ring + stage * stage_bytes + kQA, &q_map, k * kQCols, tok_tile * a.n + rank * (a.n / 2), s32(&s_full[stage]));
            };
            int issued = 0, stage = 0;
            uint32_t parity = 1;  // of the wait for a stage that is being used again
            bool ok = true;
            for (int tile = cluster; tile < n_tiles && ok; tile += n_clusters) {
                int row_tile, tok_tile;
                place(tile, row_tile, tok_tile);
                int k = k0;
                if (issued == 0) {
                    // Weights are in place before the launch (where they may not be, the caller has turned overlap off); what the kernel before this one in the stream makes, the activations, is waited for.
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
            // D s32, A and B s8, K-major
            const uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(a.n >> 3) << 17) | (static_cast<uint32_t>(GROUP * kQRows >> 4) << 24);
            int stage = 0, done = 0;
            uint32_t parity = 0;
            bool ok = true;
            for (int tile = cluster; tile < n_tiles && ok; tile += n_clusters, ++done) {
                const int buf = SPLIT ? 0 : done & 1;
                if (rank == 0 && done >= 2) {
                    ok = wait<PAIR>(s32(&s_acc_empty[buf]), ((done >> 1) - 1) & 1, failed);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                }
                const uint32_t acc = tmem + buf * a.acc_cols;
                for (int k = k0; k < k1; ++k) {
                    const uint32_t full = s32(&s_full[stage]);
                    ok = !stalled(part, k - k0) && (PAIR && rank == 0 ? wait<true>(full, parity, failed) : wait<false>(full, parity, failed));
                    if (!ok) break;
                    if (rank == 0) {
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint64_t w_desc = tile_desc(ring + stage * stage_bytes), q_desc = tile_desc(ring + stage * stage_bytes + kQA);
#pragma unroll
                        for (int j = 0; j < kQCols / 32; ++j) mma_i8<PAIR>(acc, w_desc + 2 * j, q_desc + 2 * j, idesc, (k > k0 || j > 0) ? 1u : 0u);
                        commit<PAIR>(s32(&s_empty[stage]), static_cast<uint32_t>(part));
                    } else {
                        arrive_in(in_block(full, static_cast<int>(leader)));
                    }
                    if (++stage == a.stages) stage = 0, parity ^= 1;
                }
                if (ok && rank == 0) commit<PAIR>(s32(&s_acc_full[buf]), static_cast<uint32_t>(part));
            }
        }
        __syncwarp();
    }

    if constexpr (!SPLIT) {
        if (warp >= 4) {
            const int lanes = warp & 3, half = (warp - 4) >> 2;  // (a warp may read the 32 lanes (warp % 4) * 32 onwards)
            asm volatile("griddepcontrol.wait;" ::: "memory");
            int done = 0;
            bool ok = true;  // (once a wait has given up the writers go on to the end without writing: they meet at a barrier for every tile)
            for (int tile = cluster; tile < n_tiles; tile += n_clusters, ++done) {
                int row_tile, tok_tile;
                place(tile, row_tile, tok_tile);
                const int buf = done & 1, row = (row_tile * GROUP + rank) * kQRows + lanes * 32 + lane;
                const float w_scale = row < a.rows ? __ldg(a.w_scales + row) : 0.0f;
                fetch_scales(a, tok_tile * a.n, s_scales[buf]);
                ok = ok && warp_wait(s32(&s_acc_full[buf]), (done >> 1) & 1, failed);
                if (!ok) continue;
                if (tile + n_clusters >= n_tiles) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t at = tmem + buf * a.acc_cols + (static_cast<uint32_t>(lanes * 32) << 16);
                int v[16], next[16];
                load_sums(at + half * 16, v);  // (pairs' tiles and those of more than 16 rows are wide enough; of 16 the second warp reads and writes nothing)
#pragma unroll 1
                for (int c = half * 16; c < a.n; c += 32) {
                    loaded();
#pragma unroll
                    for (int j = 0; j < 16; ++j) next[j] = v[j];
                    if (c + 32 < a.n) load_sums(at + c + 32, v);  // (on its way while these are written)
                    write_any(a, next, row, tok_tile * a.n + c, w_scale, s_scales[buf] + c);
                }
                loaded();
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    if constexpr (PAIR) arrive_in(in_block(s32(&s_acc_empty[buf]), static_cast<int>(leader)));
                    else bar_arrive(s32(&s_acc_empty[buf]));
                }
            }
        }
    } else {
        // One tile; its sums go, 8 columns of 32 lanes at a time, to the block that writes them: unit u to part u % split.
        const int lanes = warp & 3, half = (warp - 4) >> 2;
        const uint32_t at = tmem + (static_cast<uint32_t>(lanes * 32) << 16);
        int row_tile, tok_tile;
        place(cluster, row_tile, tok_tile);
        const int row = (row_tile * GROUP + rank) * kQRows + lanes * 32 + lane;
        float w_scale = 0.0f;
        bool whole = false;  // else nothing is sent, and who waits for it gives up too
        if (warp >= 4) {
            if (row < a.rows) w_scale = __ldg(a.w_scales + row);
            asm volatile("griddepcontrol.wait;" ::: "memory");
            fetch_scales(a, tok_tile * a.n, s_scales[0]);
            whole = warp_wait(s32(&s_acc_full[0]), 0, failed);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        }
        const uint32_t sums = s32(&s_sums), room = ring + a.exchange;
        const bool own_room = a.exchange != 0;
        if (!own_room) cluster_sync();  // every block's MMAs are done with its stages, where the sums go
        if (warp >= 4) {
            for (int c = half; c < a.n / 8; c += 2) {
                const int unit = c * 4 + lanes, owner = unit % a.split;
                if (owner == part || !whole) continue;
                int v[8];
                load_sums(at + c * 8, v);
                loaded();
                // stores that count their bytes on a barrier of the block that they go to
                const uint32_t to = in_block(room + ((unit / a.split) * (a.split - 1) + (part < owner ? part : part - 1)) * 1024 + lane * 16, owner * GROUP + rank);
                const uint32_t bar = in_block(sums, owner * GROUP + rank);
                asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(bar)
                             : "memory");
                asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(to + 512), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(bar)
                             : "memory");
            }
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // (its other half is at the end: until then others may still send)
        if (warp >= 4) {
            asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
            const int units = a.n / 2, mine = units / a.split + (part < units % a.split ? 1 : 0);  // of this block
            if (warp == 4 && lane == 0) expect(sums, static_cast<uint32_t>(mine * (a.split - 1)) * 1024);
            const bool ok = wait<true>(sums, 0, failed);  // (by every lane: it reads what others have stored)
            __syncwarp();
            for (int c = half; c < a.n / 8; c += 2) {
                const int unit = c * 4 + lanes;
                if (unit % a.split != part) continue;
                int v[8];
                load_sums(at + c * 8, v);
                loaded();
                for (int p = 0; p < a.split - 1; ++p) {
                    const uint32_t from = room + ((unit / a.split) * (a.split - 1) + p) * 1024 + lane * 16;
                    const uint4 x = lds128u(from), z = lds128u(from + 512);
                    v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w, v[4] += z.x, v[5] += z.y, v[6] += z.z, v[7] += z.w;
                }
                if (ok && whole && !*failed) write_any(a, v, row, tok_tile * a.n + c * 8, w_scale, s_scales[0] + c * 8);
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
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(a.tmem_cols) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(a.tmem_cols) : "memory");
        if (lane == 0 && s_failed) atomicExch(a.status, kStatusWaitExpired);
    }
}

template <bool PAIR, bool SPLIT>
struct Variant {
    static constexpr int smem(bool half) { return (half ? kQHalfRing : kQRing) + 1024; }
    static constexpr int kGroup = PAIR ? 2 : 1;
    static constexpr auto kKernel = qmm_i8_kernel<PAIR, SPLIT>;
    static void configure(cudaLaunchConfig_t &cfg, cudaLaunchAttribute *attr, int clusters, int split, bool half, bool overlap, cudaStream_t stream) {
        cfg.gridDim = dim3(static_cast<unsigned>(clusters * split * kGroup));
        cfg.blockDim = dim3(kQThreads);
        cfg.dynamicSmemBytes = smem(half);
        cfg.stream = stream;
        cfg.attrs = attr;
        cfg.numAttrs = launch_attributes(attr, overlap, split * kGroup);
    }
    // clusters that fit on the GPU at once, one block per SM (cached; one device per process), 0 if the kernel cannot run
    static int clusters(int split) {
        static int cached[kQMaxSplit + 1] = {};
        if (cached[split] == 0) {
            int n = 0;
            cudaLaunchConfig_t cfg{};
            cudaLaunchAttribute attr[2];
            configure(cfg, attr, 1024, split, false, true, nullptr);
            if (cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem(false)) != cudaSuccess || cudaOccupancyMaxActiveClusters(&n, kKernel, &cfg) != cudaSuccess) {
                (void)cudaGetLastError();
                n = 0;
            }
            cached[split] = n > 0 ? n : -1;
        }
        return cached[split] < 0 ? 0 : cached[split];
    }
    static cudaError_t launch(const CUtensorMap &w, const CUtensorMap &q, const QmmTc &a, bool overlap, cudaStream_t stream) {
        const int fit = clusters(a.split), tiles = a.row_tiles * a.tok_tiles;
        if (fit == 0) return cudaErrorInvalidConfiguration;
        cudaLaunchConfig_t cfg{};
        cudaLaunchAttribute attr[2];
        configure(cfg, attr, SPLIT ? tiles : (tiles < fit ? tiles : fit), a.split, a.half_sm != 0, overlap, stream);
        return cudaLaunchKernelEx(&cfg, kKernel, w, q, a);
    }
};

}  // namespace

cudaError_t launch_qmm_i8(const QmmI8Args &in, cudaStream_t stream) {
    QmmTc a{};
    a.w_scales = in.w_scales;
    a.q_scales = in.q_scales;
    a.y = in.y;
    a.status = in.status;
    a.rows = in.rows;
    a.ntok = in.ntok;
    a.n_k = (in.cols + kQCols - 1) / kQCols;
    a.y_elem = in.y_elem;
    a.add = in.add;
    const bool pair = in.ntok > 256;
    const int group = pair ? 2 : 1, step = pair ? 32 : 16;
    a.tok_tiles = (in.ntok + kQMaxN - 1) / kQMaxN;
    a.n = ((in.ntok + a.tok_tiles - 1) / a.tok_tiles + step - 1) / step * step;
    a.tok_tiles = (in.ntok + a.n - 1) / a.n;
    a.row_tiles = (in.rows + group * kQRows - 1) / (group * kQRows);
    // As many parts of the columns as leave every cluster room beside the others, of two stages at least.
    a.split = 1;
    const int tiles = a.row_tiles * a.tok_tiles;
    for (int split = 2; split <= (pair ? kQMaxSplit / 2 : kQMaxSplit) && a.n_k >= 2 * split; ++split)
        if (tiles <= (pair ? Variant<true, true>::clusters(split) : Variant<false, true>::clusters(split))) a.split = split;
    const bool brief = a.n_k <= 8 * a.split;  // a few stages for each block: what counts is how soon it begins and ends
    a.half_sm = !pair && a.n <= (brief ? 80 : 32);
    a.b_bytes = a.n / group * kQCols;
    // Sums have memory of their own where that costs no stage or the stages are few, else they go where the stages were, one barrier of the cluster later.
    const int ring = a.half_sm ? kQHalfRing : kQRing, units = a.n / 2, room = a.split > 1 ? (units + a.split - 1) / a.split * (a.split - 1) * 1024 : 0;
    a.stages = ring / (kQA + a.b_bytes);
    const int beside = (ring - room) / (kQA + a.b_bytes);
    if (a.split > 1 && (beside == a.stages || (brief && beside >= 3))) a.exchange = ring - room, a.stages = beside;
    if (a.stages > kQMaxStages) a.stages = kQMaxStages;
    a.acc_cols = 32;
    while (a.acc_cols < a.n) a.acc_cols *= 2;
    a.tmem_cols = (a.split > 1 ? 1 : 2) * a.acc_cols;
    CUtensorMap w, q;
    cudaError_t err = encode_rows(&w, in.w, in.cols, in.w_pitch, in.rows, kQRows);
    if (err == cudaSuccess) err = encode_rows(&q, in.q, in.cols, i8_pitch(in.cols), in.ntok, a.n / group);
    if (err != cudaSuccess) return err;
    if (pair) return a.split > 1 ? Variant<true, true>::launch(w, q, a, in.overlap, stream) : Variant<true, false>::launch(w, q, a, in.overlap, stream);
    return a.split > 1 ? Variant<false, true>::launch(w, q, a, in.overlap, stream) : Variant<false, false>::launch(w, q, a, in.overlap, stream);
}

}  // namespace vqm
