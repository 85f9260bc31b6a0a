// Product of e4m3 activations (a scale for each 128 columns of a row) and e4m3 weights (a scale for each block of 128 x 128) on the 5th-generation tensor
// cores:  y[t][r] = sum_b sx[b][t] sw[r / 128][b] sum_{k in block b} q[t][k] W[r][k].
//
// A stage of the ring is a block of 128 columns of both operands, by TMA.  Its products are summed by tcgen05.mma (kind::f8f6f4) into an accumulator of its own in
// tensor memory; the writers read that, and add it times the two scales to sums in registers, all of them fp32.  (An accumulator cannot be scaled where it is, and scales in
// the operands would have to be powers of two.)  The scales' product is fp32: in two factors where that does not hold it, which the header leaves open, was 3 to 5 % slower for all
// calls, and 11 for 24 rows of 5120 x 17408.  With two or four accumulators the next blocks are multiplied meanwhile.
//   warp 0      one thread issues the copies
//   warp 1      one thread issues the MMAs (in the second block of a pair: passes "full" on to the first)
//   warp 2      tensor memory
//   warps 4-11  sums and outputs: two warps for each 32 lanes of tensor memory, each half of the columns
// Up to 64 activation rows: the weight rows are the lanes, the activation rows the columns (16, 32 or 64).  A lane's weight scale is the block's, the activation scales
// are one for each column, by shared memory.
// TURNED, more: the activation rows are the lanes, 128 weight rows the columns, and a lane needs one factor for all of its columns.  (With the weight rows in the lanes
// it would need 128 different ones, which shared memory gives in twice the time of the MMAs.)  Outputs go out by TMA, where rows are multiples of 16 bytes.
// PAIR, many rows: two blocks of a cluster multiply 256 activation rows by 256 weight rows together (cta_group::2), each half of the weight rows by itself, so
// that four accumulators are in turn.
// SPLIT (few tiles): the blocks, or pairs, of a cluster share the columns of a tile, and exchange their sums by st.async, so that no memory of the runtime is involved.
//
// What bounds it.  Few rows: memory.  17408 x 5120, one launch behind the other: 1 row 17.7 us (5.0 TB/s), 16 18.0, 32 19.9, 64 21.3, of which 3 to 4 are the start and the
// end of a launch; among others 13.5 (6.6 TB/s).  Many: the writers, then power.  A pair's MMAs take 512 cycles for a block of columns, its writers 626 without a wait
// (each warp eight loads of 16 columns and 64 fused multiply-adds of two sums), and the hand-over between the two makes that 790: 512 rows 46 to 50 us, 2048 163 to
// 180, 4096 312 to 317 (2.3 PFLOP/s; 267 with weights of zeros, which keep the clock up).  Neither polling without a suspend time, nor one thread for the MMAs of
// both halves, nor other shares of the registers (208 and 232 of a writer) was faster.
//
// Every wait is bounded: on expiry the block records a status code and everybody falls through to the end.
#include <cuda.h>
#include <cuda_fp16.h>

#include <climits>

#include "vqm_kernels.h"
#include "vqm_tiles8.cuh"

namespace vqm {
namespace {

constexpr int kRows = 128;                  // rows of a block's first operand, the lanes of tensor memory
constexpr int kABytes = kRows * kQCols;     // of a stage
constexpr int kMaxStages = 12, kMaxCluster = 8;
constexpr int kRing = 216 * 1024, kHalfRing = 106 * 1024, kTurnedRing = 160 * 1024, kBox = 4096, kStaging = 2 * kBox;  // (a warp's, for outputs on their way)
constexpr int kWriters = 8, kThreads = 128 + 32 * kWriters;
// Registers of a thread: a pair's writers hold 128 sums and two sets of 16 that come from tensor memory.  The shares add up to what the block is launched with.
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
    int tile_out;                      // TURNED: outputs go out by TMA
};
template <bool TURNED>
struct Maps {
    CUtensorMap w, q;
};
template <>
struct Maps<true> {
    CUtensorMap w, q, y;
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
// A pair's copies, whichever block they go to, are counted on a barrier of the first.
__device__ __forceinline__ void copy_tile_of_pair(uint32_t to, const CUtensorMap *map, int x, int row, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(to), "l"(map), "r"(x), "r"(row), "r"(bar)
                 : "memory");
}
// Tensor memory has been read (and a fence says so): nothing else is handed over, so that loads on their way are not waited for.
__device__ __forceinline__ void arrive_relaxed(uint32_t cluster_addr) { asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory"); }
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

__device__ __forceinline__ void add_scaled(float &s0, float &s1, uint32_t x, uint32_t y, float a, float b) {
    asm("{\n\t.reg .b64 v, c, d;\n\tmov.b64 v, {%2, %3};\n\tmov.b64 c, {%4, %5};\n\tmov.b64 d, {%0, %1};\n\tfma.rn.f32x2 d, v, c, d;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "+f"(s0), "+f"(s1)
        : "r"(x), "r"(y), "f"(a), "f"(b));
}

// Whether the barrier's phase is over, without waiting.
__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}

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
__device__ __forceinline__ void write8_any(const QmmF8 &a, long long at, long long stride, int left, bool add, float (&v)[8]) {
    if (a.y_elem == 2) write8(static_cast<__half *>(a.y) + at, stride, left, add, v);
    else write8(static_cast<float *>(a.y) + at, stride, left, add, v);
}

// Eight outputs that lie side by side, of an activation row; rows begin on four outputs.  What they are added to comes first, as it is.
template <typename Y>
__device__ __forceinline__ void read8_along(const Y *y, int row, int rows, float (&was)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (row + 4 * i < rows) {
            if constexpr (sizeof(Y) == 4) {
                const float4 w = *reinterpret_cast<const float4 *>(y + row + 4 * i);
                was[4 * i] = w.x, was[4 * i + 1] = w.y, was[4 * i + 2] = w.z, was[4 * i + 3] = w.w;
            } else {
                const float2 w = *reinterpret_cast<const float2 *>(y + row + 4 * i);
                was[4 * i] = w.x, was[4 * i + 1] = w.y;
            }
        }
}
template <typename Y>
__device__ __forceinline__ void write8_along(Y *y, int row, int rows, bool add, const float (&was)[8], float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (row + 4 * i >= rows) break;
        float four[4] = {v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
        if (add) {
            if constexpr (sizeof(Y) == 4) {
#pragma unroll
                for (int e = 0; e < 4; ++e) four[e] += was[4 * i + e];
            } else {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t bits = __float_as_uint(was[4 * i + e]);
                    const float2 w = __half22float2(*reinterpret_cast<const __half2 *>(&bits));
                    four[2 * e] += w.x, four[2 * e + 1] += w.y;
                }
            }
        }
        put4(y + row + 4 * i, four);
    }
}
// Rows that do not: eight outputs of each of 32 activation rows, which lie in shared memory, by the whole warp, four rows at a time.  (A store of two bytes in each of 32 rows
// takes as long as one of 16: 1001 x 4999 with 177 rows, fp16, 12.2 us that way and 10.7.)
__device__ __forceinline__ void write8_odd(const QmmF8 &a, uint32_t room, int tok0, int row) {
    const int lane = threadIdx.x & 31, t = tok0 + (lane >> 3), col = row + (lane & 7);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v[i]) : "r"(room + i * 128 + lane * 4));
    if (col < a.rows) write8_any(a, static_cast<long long>(t) * a.rows + col, 4ll * a.rows, (a.ntok - t + 3) / 4, a.add != 0, v);
}

// 32 activation rows (of the lanes) by 32 weight rows (of a lane's values), turned in shared memory so that what is written together lies together.  `room`: a
// warp's 4 KB, rows of 128 bytes whose 16-byte pieces are exchanged against bank conflicts.
template <typename Y>
__device__ __forceinline__ void write_turned(const QmmF8 &a, uint32_t room, const float *sums, int tok0, int row0) {
    const int lane = threadIdx.x & 31, piece = lane & 7, row = row0 + piece * 4;
    Y *const y = static_cast<Y *>(a.y), *const at = y + static_cast<long long>(tok0 + (lane >> 3)) * a.rows + row;
    const bool whole = a.rows % 4 == 0;  // (buffers are 16-byte aligned)
    float was[8][4];                     // on its way before anything else
    if (whole && a.add && row < a.rows)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (tok0 + i * 4 + (lane >> 3) < a.ntok) get4(at + i * 4ll * a.rows, was[i]);
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t to = room + lane * 128 + ((j ^ (lane & 7)) * 16);
        asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(sums[4 * j]), "f"(sums[4 * j + 1]), "f"(sums[4 * j + 2]), "f"(sums[4 * j + 3]) : "memory");
    }
    __syncwarp();
    if (whole) {
        if (row < a.rows) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int t = i * 4 + (lane >> 3);
                const uint4 w = lds128u(room + t * 128 + ((piece ^ (t & 7)) * 16));
                float v[4] = {__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w)};
                if (a.add)
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] += was[i][e];
                if (tok0 + t < a.ntok) put4(at + i * 4ll * a.rows, v);
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

// The same by TMA, a box of 128 bytes of 32 activation rows at a time; two boxes of a warp in turn.
template <typename Y, int CW>
__device__ __forceinline__ void write_boxes(const QmmF8 &a, const CUtensorMap *map, uint32_t room, uint32_t &turn, const float *sums, int tok0, int row0) {
    constexpr int COLS = 128 / sizeof(Y);
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int b = 0; b < CW / COLS; ++b) {
        const uint32_t box = room + (turn++ & 1) * kBox;
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");  // (the store before the last one has read its box)
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t to = box + lane * 128 + ((j ^ (lane & 7)) * 16);
            if constexpr (sizeof(Y) == 4) {
                const float *v = sums + b * 32 + 4 * j;
                asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]) : "memory");
            } else {
                uint32_t h[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const __half2 v = __floats2half2_rn(sums[b * 64 + 8 * j + 2 * i], sums[b * 64 + 8 * j + 2 * i + 1]);
                    h[i] = *reinterpret_cast<const uint32_t *>(&v);
                }
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
            // (what is beyond the last row or column is not written; no box begins there)
            if (tok0 < a.ntok && row0 + b * COLS < a.rows)
                asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(row0 + b * COLS), "r"(tok0), "r"(box) : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
    }
}

// CW: columns of tensor memory that a writer warp reads
__host__ __device__ constexpr bool turned(int cw) { return cw >= 64; }  // the lanes are activation rows
__host__ __device__ constexpr bool paired(int cw) { return cw == 128; }
template <int CW, bool SPLIT>
__global__ void __launch_bounds__(kThreads, CW <= 16 ? 2 : 1) qmm_f8_kernel(const __grid_constant__ Maps<turned(CW)> maps, const QmmF8 a) {
    constexpr bool PAIR = paired(CW), TURNED = turned(CW);
    constexpr int GROUP = PAIR ? 2 : 1, N = 2 * CW, BUFS = PAIR ? 2 : 4, TMEM = N * BUFS;
    constexpr int HALVES = PAIR ? 2 : 1;  // parts of an accumulator that are multiplied, and handed on, by themselves
    extern __shared__ uint8_t ring_raw[];
    __shared__ __align__(8) uint64_t s_full[kMaxStages], s_empty[kMaxStages], s_acc_full[HALVES][BUFS], s_acc_empty[HALVES][BUFS], s_sums[kWriters];
    __shared__ __align__(16) float s_scales[TURNED ? 1 : kWriters][2][TURNED ? 4 : CW];
    __shared__ uint32_t s_tmem;
    __shared__ int s_failed;
    const uint32_t ring = (s32(ring_raw) + 1023u) & ~1023u;  // (the swizzle works on address bits)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t in_cluster = 0;
    if constexpr (PAIR || SPLIT) asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(in_cluster));
    const int rank = PAIR ? static_cast<int>(in_cluster & 1u) : 0, part = SPLIT ? static_cast<int>(in_cluster) / GROUP : 0;  // place in the pair, share of the columns
    const uint32_t leader = in_cluster & ~1u;
    const int cluster = static_cast<int>(blockIdx.x) / (GROUP * a.split), n_clusters = static_cast<int>(gridDim.x) / (GROUP * a.split);
    const int k0 = SPLIT ? part * a.n_k / a.split : 0, k1 = SPLIT ? (part + 1) * a.n_k / a.split : a.n_k;
    const int n_tiles = a.row_tiles * a.tok_tiles;
    const uint32_t stage_bytes = kABytes + a.b_bytes;

    if (threadIdx.x == 0) {
        for (int s = 0; s < a.stages; ++s) {
            bar_init(s32(&s_full[s]), 1);  // (a pair's: the first block's)
            bar_init(s32(&s_empty[s]), HALVES);
        }
        for (int h = 0; h < HALVES; ++h)
            for (int b = 0; b < BUFS; ++b) {
                bar_init(s32(&s_acc_full[h][b]), 1);
                bar_init(s32(&s_acc_empty[h][b]), kWriters / HALVES * GROUP);
            }
        for (int w = 0; w < kWriters; ++w) bar_init(s32(&s_sums[w]), 1);
        s_failed = 0;
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
        if constexpr (!TURNED) {
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
                const uint32_t full0 = PAIR ? in_block(s32(&s_full[0]), static_cast<int>(leader)) : s32(&s_full[0]);
                const uint32_t to0 = PAIR ? in_block(ring, static_cast<int>(in_cluster)) : ring;
                auto copy_w = [&](int stage, int k, int row_tile) {
                    if constexpr (PAIR) {  // 64 rows of each half
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            copy_tile_of_pair(to0 + stage * stage_bytes + kABytes + h * (kABytes / 2), &maps.w, k * kQCols, (row_tile * 2 + h) * kRows + rank * (kRows / 2), full0 + stage * 8);
                    } else {
                        copy_tile(to0 + stage * stage_bytes + (TURNED ? kABytes : 0), &maps.w, k * kQCols, row_tile * kRows, full0 + stage * 8);
                    }
                };
                auto copy_q = [&](int stage, int k, int tok_tile) {
                    if constexpr (PAIR) copy_tile_of_pair(to0 + stage * stage_bytes, &maps.q, k * kQCols, (tok_tile * GROUP + rank) * kRows, full0 + stage * 8);
                    else copy_tile(to0 + stage * stage_bytes + (TURNED ? 0 : kABytes), &maps.q, k * kQCols, tok_tile * kRows, full0 + stage * 8);
                };
                auto expect_stage = [&](int stage) {
                    if (rank == 0) expect(s32(&s_full[stage]), GROUP * stage_bytes);
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
                            expect_stage(i);
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
                        expect_stage(stage);
                        copy_w(stage, k, row_tile);
                        copy_q(stage, k, tok_tile);
                        ++issued;
                        if (++stage == a.stages) stage = 0, parity ^= 1;
                    }
                }
                // The last copies land before the block goes on to its end, or in a cluster says that others may: whatever waits have given up, none comes to memory that is
                // somebody else's by then.  In the second block of a pair, whose copies are counted in the first, the MMAs' having read them says so; where those have given
                // up, the time that this takes to give up too.
                const uint32_t landed = rank == 0 ? s32(&s_full[0]) : s32(&s_empty[0]);
                int left = 1 << 16;
                for (int last = max(0, issued - a.stages); last < issued; ++last)
                    while (!bar_test(landed + last % a.stages * 8, (last / a.stages) & 1) && --left > 0) __nanosleep(64);
            }
            __syncwarp();
        } else if (warp == 1 || (PAIR && warp == 3)) {
            if (rank == 0 && tc::elect_one()) {
                const int part_of = warp >> 1;  // the half that this warp multiplies
                // D fp32, A and B e4m3, K-major
                const uint32_t idesc = (1u << 4) | (static_cast<uint32_t>(N / HALVES >> 3) << 17) | (static_cast<uint32_t>(GROUP * kRows >> 4) << 24);
                int stage = 0, done = 0;
                uint32_t parity = 0;
                bool ok = true;
                for (int tile = cluster; tile < n_tiles && ok; tile += n_clusters) {
                    for (int k = k0; k < k1; ++k, ++done) {
                        const uint32_t full = s32(&s_full[stage]);
                        const int buf = done % BUFS;
                        ok = !stalled(part, done) && wait<false>(full, parity, failed);
                        if (ok && done >= BUFS) ok = wait<false>(s32(&s_acc_empty[part_of][buf]), (done / BUFS - 1) & 1, failed);
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint64_t a_desc = tile_desc(ring + stage * stage_bytes), b_desc = tile_desc(ring + stage * stage_bytes + kABytes + part_of * (kABytes / 2));
#pragma unroll
                        for (int j = 0; j < kQCols / 32; ++j) mma_f8<PAIR>(tmem + buf * N + part_of * CW, a_desc + 2 * j, b_desc + 2 * j, idesc, j > 0 ? 1u : 0u);
                        commit<PAIR>(s32(&s_acc_full[part_of][buf]), static_cast<uint32_t>(part));
                        commit<PAIR>(s32(&s_empty[stage]), static_cast<uint32_t>(part));
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
        const int writer = warp - 4, lanes = warp & 3, half = writer >> 2, part_of = PAIR ? half : 0;  // (a warp may read the 32 lanes (warp % 4) * 32 onwards)
        asm volatile("griddepcontrol.wait;" ::: "memory");
        bool ok = true;
        float sums[CW];
        uint32_t turn = 0, box_turn = 0;  // blocks of columns, boxes of outputs so far
        bool ready = false;               // the accumulator of this turn is known to be there
        const uint32_t emptied = PAIR ? in_block(s32(&s_acc_empty[part_of][0]), static_cast<int>(leader)) : s32(&s_acc_empty[0][0]);
        int row0 = 0, tok0 = 0;  // of this lane's outputs: TURNED: activation row tok0, weight rows from row0 on; else weight row row0, activation rows from tok0 on
        for (int tile = cluster; tile < n_tiles; tile += n_clusters) {
            int row_tile, tok_tile;
            place(tile, row_tile, tok_tile);
#pragma unroll
            for (int j = 0; j < CW; ++j) sums[j] = 0.0f;
            if constexpr (TURNED) {
                // (what is beyond the last row takes the last one's scales)
                const float *sx = a.q_scales + min((tok_tile * GROUP + rank) * kRows + lanes * 32 + lane, a.ntok - 1) + k0 * a.q_scale_pitch;
                const float *sw = a.w_scales + static_cast<size_t>(min(PAIR ? row_tile * 2 + half : row_tile, (a.rows - 1) / kF8Block)) * a.n_k + k0;
                float x_next = *sx, w_next = __ldg(sw);  // on their way one block ahead
#pragma unroll 1
                for (int left = k1 - k0; left > 0; --left, ++turn) {
                    const int buf = turn % BUFS;
                    if (!ready) ok &= wait<false>(s32(&s_acc_full[part_of][buf]), (turn / BUFS) & 1, failed);  // (no way out of the loop: the sums would be copied)
                    __syncwarp();
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t at = tmem + buf * N + half * CW + (static_cast<uint32_t>(lanes * 32) << 16);
                    constexpr int PW = 16;  // columns of one load
                    uint32_t v[2][PW];
                    load_sums<PW>(at, v[0]);
                    load_sums<PW>(at + PW, v[1]);
                    const float scale = x_next * w_next;
                    if (left > 1) {
                        sx += a.q_scale_pitch, ++sw;
                        x_next = *sx, w_next = __ldg(sw);
                    }
#pragma unroll
                    for (int p = 0; p < CW / PW; ++p) {
                        if (p % 2 == 0) loaded();
                        if (p + 2 == CW / PW) {  // the accumulator may be used again, and whether the next one is there shows while these are added
                            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                            __syncwarp();
                            if (lane == 0) {
                                if constexpr (PAIR) arrive_relaxed(emptied + buf * 8);
                                else bar_arrive(emptied + buf * 8);
                            }
                            ready = bar_test(s32(&s_acc_full[part_of][(turn + 1) % BUFS]), ((turn + 1) / BUFS) & 1);
                        }
#pragma unroll
                        for (int j = 0; j < PW; j += 2) add_scaled(sums[p * PW + j], sums[p * PW + j + 1], v[p & 1][j], v[p & 1][j + 1], scale, scale);
                        if (p + 2 < CW / PW) load_sums<PW>(at + (p + 2) * PW, v[p & 1]);
                    }
                }
                place(tile, row_tile, tok_tile);
                tok0 = (tok_tile * GROUP + rank) * kRows + lanes * 32 + lane;
                row0 = row_tile * 2 * CW + half * CW;
            } else {
                row0 = row_tile * kRows + lanes * 32 + lane;
                tok0 = half * CW;
                const bool has_x = lane < CW && tok0 + lane < a.ntok;
                const float *sx = a.q_scales + tok0 + lane + k0 * a.q_scale_pitch, *sw = a.w_scales + static_cast<size_t>(row_tile) * a.n_k + k0;
                float x_next = has_x ? *sx : 0.0f, w_next = __ldg(sw);
#pragma unroll 1
                for (int left = k1 - k0; left > 0; --left, ++turn) {
                    const int buf = turn % BUFS;
                    float *scales = s_scales[writer][buf & 1];
                    if (lane < CW) scales[lane] = x_next * w_next;
                    __syncwarp();  // (and nobody reads what the next block but one replaces)
                    if (left > 1) {
                        sx += a.q_scale_pitch, ++sw;
                        if (has_x) x_next = *sx;
                        w_next = __ldg(sw);
                    }
                    if (!ready) ok &= wait<false>(s32(&s_acc_full[0][buf]), (turn / BUFS) & 1, failed);
                    __syncwarp();
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    uint32_t v[CW];
                    load_sums<CW>(tmem + buf * N + half * CW + (static_cast<uint32_t>(lanes * 32) << 16), v);
                    loaded();
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) bar_arrive(emptied + buf * 8);
                    ready = bar_test(s32(&s_acc_full[0][(turn + 1) % BUFS]), ((turn + 1) / BUFS) & 1);
#pragma unroll
                    for (int j = 0; j < CW; j += 4) {
                        const float4 s = *reinterpret_cast<const float4 *>(scales + j);
                        add_scaled(sums[j], sums[j + 1], v[j], v[j + 1], s.x, s.y);
                        add_scaled(sums[j + 2], sums[j + 3], v[j + 2], v[j + 3], s.z, s.w);
                    }
                }
            }
            if constexpr (!SPLIT) {
                if (tile + n_clusters >= n_tiles) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
                if (!__all_sync(0xFFFFFFFFu, ok)) continue;  // (once a wait has given up the writers go on to the end without writing)
                if constexpr (TURNED) {
                    const uint32_t room = ring + kTurnedRing + writer * kStaging;
                    if (a.tile_out) {
                        if (a.y_elem == 2) write_boxes<__half, CW>(a, &maps.y, room, box_turn, sums, tok0 - lane, row0);
                        else write_boxes<float, CW>(a, &maps.y, room, box_turn, sums, tok0 - lane, row0);
                    } else {
#pragma unroll
                        for (int p = 0; p < CW / 32; ++p) {
                            if (a.y_elem == 2) write_turned<__half>(a, room, sums + p * 32, tok0 - lane, row0 + p * 32);
                            else write_turned<float>(a, room, sums + p * 32, tok0 - lane, row0 + p * 32);
                        }
                    }
                } else if (row0 < a.rows) {
#pragma unroll
                    for (int c = 0; c < CW / 8; ++c) {
                        float v[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = sums[8 * c + j];
                        write8_any(a, static_cast<long long>(tok0 + 8 * c) * a.rows + row0, a.rows, a.ntok - tok0 - 8 * c, a.add != 0, v);
                    }
                }
            }
        }
        if constexpr (TURNED && !SPLIT)
            if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        if constexpr (SPLIT) {
            // One tile; its sums go, 8 columns of 32 lanes at a time (a unit), to the block that writes them, and there to the same warp.
            const uint32_t room = ring + a.exchange, bar = s32(&s_sums[writer]);
            const int of_column = (kWriters + a.split - 1) / a.split;  // units of 8 columns that a block may have
            const int first_owner = writer % a.split;
            auto free_room = [&](int c) { return room + static_cast<uint32_t>((c * of_column + writer / a.split) * (a.split - 1)) * 1024; };  // (once this warp has read what came)
            auto room_of = [&](int c, int from, int owner) { return room + static_cast<uint32_t>((c * of_column + writer / a.split) * (a.split - 1) + (from < owner ? from : from - 1)) * 1024 + lane * 16; };
            if (a.exchange == 0) cluster_sync();  // every block's MMAs are done with its stages, where the sums go (in one that has given up, no copy is on its way)
            const bool whole = __all_sync(0xFFFFFFFFu, ok);  // else nothing is sent, and who waits for it gives up too
            int mine = 0, next = first_owner;
            auto owner_next = [&] {  // of unit 0, 1, ...
                const int owner = next;
                next = next + 1 == a.split ? 0 : next + 1;
                return owner;
            };
#pragma unroll
            for (int c = 0; c < CW / 8; ++c) {
                const int owner = owner_next();
                if (owner == part) {
                    ++mine;
                    continue;
                }
                if (!whole) continue;
                // stores that count their bytes on a barrier of the block that they go to
                const int block = owner * GROUP + rank;
                const uint32_t to = in_block(room_of(c, part, owner), block), there = in_block(bar, block);
                asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(to), "f"(sums[8 * c + 0]), "f"(sums[8 * c + 1]), "f"(sums[8 * c + 2]), "f"(sums[8 * c + 3]), "r"(there)
                             : "memory");
                asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(to + 512), "f"(sums[8 * c + 4]), "f"(sums[8 * c + 5]), "f"(sums[8 * c + 6]), "f"(sums[8 * c + 7]), "r"(there)
                             : "memory");
            }
            // What outputs are added to is on its way while the others' sums are waited for: a unit's is kept where the sums of its neighbour were (the other one of two, which
            // has another owner and has been sent).
            [[maybe_unused]] float onto[TURNED ? 1 : CW];
            if (a.add) {
                next = first_owner;
#pragma unroll
                for (int c = 0; c < CW / 8; ++c) {
                    if (owner_next() != part) continue;
                    if constexpr (TURNED) {
                        float was[8] = {};
                        if (a.rows % 4 == 0 && tok0 < a.ntok) {
                            if (a.y_elem == 2) read8_along(static_cast<const __half *>(a.y) + static_cast<long long>(tok0) * a.rows, row0 + 8 * c, a.rows, was);
                            else read8_along(static_cast<const float *>(a.y) + static_cast<long long>(tok0) * a.rows, row0 + 8 * c, a.rows, was);
                        }
#pragma unroll
                        for (int j = 0; j < 8; ++j) sums[8 * (c ^ 1) + j] = was[j];
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const int t = tok0 + 8 * c + j;
                            const long long at = static_cast<long long>(t) * a.rows + row0;
                            onto[8 * c + j] = row0 >= a.rows || t >= a.ntok ? 0.0f : a.y_elem == 2 ? get(static_cast<const __half *>(a.y) + at) : get(static_cast<const float *>(a.y) + at);
                        }
                    }
                }
            }
            __syncwarp();
            asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // (its other half is at the end: until then others may still send)
            asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
            if (mine > 0) {
                if (lane == 0) expect(bar, static_cast<uint32_t>(mine * (a.split - 1)) * 1024);
                const bool there = wait<true>(bar, 0, failed);  // (by every lane: it reads what others have stored)
                __syncwarp();
                if (__all_sync(0xFFFFFFFFu, there && whole && !*failed)) {
                    next = first_owner;
#pragma unroll
                    for (int c = 0; c < CW / 8; ++c) {
                        if (owner_next() != part) continue;
                        float v[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = sums[8 * c + j];
                        for (int p = 0; p < a.split; ++p) {
                            if (p == part) continue;
                            const uint32_t from = room_of(c, p, part);
                            const uint4 x = lds128u(from), z = lds128u(from + 512);
                            v[0] += __uint_as_float(x.x), v[1] += __uint_as_float(x.y), v[2] += __uint_as_float(x.z), v[3] += __uint_as_float(x.w);
                            v[4] += __uint_as_float(z.x), v[5] += __uint_as_float(z.y), v[6] += __uint_as_float(z.z), v[7] += __uint_as_float(z.w);
                        }
                        if constexpr (TURNED) {
                            if (a.rows % 4 != 0) {
                                const uint32_t to = free_room(c) + lane * 32;
                                __syncwarp();
#pragma unroll
                                for (int i = 0; i < 8; i += 4) asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to + i * 4), "f"(v[i]), "f"(v[i + 1]), "f"(v[i + 2]), "f"(v[i + 3]) : "memory");
                            } else if (tok0 < a.ntok) {
                                float was[8];
#pragma unroll
                                for (int j = 0; j < 8; ++j) was[j] = sums[8 * (c ^ 1) + j];
                                if (a.y_elem == 2) write8_along(static_cast<__half *>(a.y) + static_cast<long long>(tok0) * a.rows, row0 + 8 * c, a.rows, a.add != 0, was, v);
                                else write8_along(static_cast<float *>(a.y) + static_cast<long long>(tok0) * a.rows, row0 + 8 * c, a.rows, a.add != 0, was, v);
                            }
                        } else {
                            if (a.add)
#pragma unroll
                                for (int j = 0; j < 8; ++j) v[j] += onto[8 * c + j];
                            if (row0 < a.rows) write8_any(a, static_cast<long long>(tok0 + 8 * c) * a.rows + row0, a.rows, a.ntok - tok0 - 8 * c, false, v);
                        }
                    }
                    if (TURNED && a.rows % 4 != 0) {
                        __syncwarp();
#pragma unroll 1
                        for (int c = (part + a.split - first_owner) % a.split; c < CW / 8; c += a.split) write8_odd(a, free_room(c), tok0 - lane, row0 + 8 * c);
                    }
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    // no block's shared or tensor memory goes away under another
    if constexpr (SPLIT) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    else if constexpr (PAIR) cluster_sync();
    if (warp == 2) {
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(TMEM) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(TMEM) : "memory");
        if (lane == 0 && s_failed) atomicExch(a.status, kStatusWaitExpired);
    }
}

// Outputs as a 2-D tensor, written in boxes of 128 bytes of 32 rows.
cudaError_t encode_outputs(CUtensorMap *map, void *y, int rows, int ntok, int elem_bytes) {
    TcEncode encode = nullptr;
    if (const cudaError_t err = tc_encoder(&encode); err != cudaSuccess) return err;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(ntok)}, strides[1] = {static_cast<cuuint64_t>(rows) * static_cast<cuuint64_t>(elem_bytes)};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(128 / elem_bytes), 32}, elem[2] = {1, 1};
    return encode(map, elem_bytes == 2 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, y, dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? cudaSuccess
               : cudaErrorInvalidValue;
}

template <int CW, bool SPLIT>
struct Variant {
    static constexpr bool PAIR = paired(CW), TURNED = turned(CW), kHalf = CW <= 16;  // two blocks per SM
    static constexpr int kGroup = PAIR ? 2 : 1, kRoom = TURNED ? kTurnedRing : kHalf ? kHalfRing : kRing;
    static constexpr int kSmem = kRoom + 1024 + (TURNED ? kWriters * kStaging : 0);
    static constexpr auto kKernel = qmm_f8_kernel<CW, SPLIT>;
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
    static cudaError_t launch(const Maps<TURNED> &maps, const QmmF8 &a, bool overlap, cudaStream_t stream) {
        const int fit = clusters(a.split), tiles = a.row_tiles * a.tok_tiles;
        if (fit == 0) return cudaErrorInvalidConfiguration;
        cudaLaunchConfig_t cfg{};
        cudaLaunchAttribute attr[2];
        configure(cfg, attr, SPLIT ? tiles : (tiles < fit ? tiles : fit), a.split, kSmem, overlap, stream);
        return cudaLaunchKernelEx(&cfg, kKernel, maps, a);
    }
};

// Parts of a tile's columns, of two blocks of columns at least, where every cluster has room beside the others.  Up to 64 activation rows: as many as that leaves
// (1024 x 5120 with 4 rows: 12.4, 8.1, 6.6, 5.9 and 5.1 us with 1, 2, 3, 4 and 8 parts).  With more, the exchange of 128 x 128 sums takes as long as 12 blocks of columns, that
// of a pair 12 us, and clusters beside which the next launch's have no room delay its beginning: as many as take least by that, at 0.27 us (0.55) for a block of columns.
// (128 rows, 1024 x 2048: 7.4, 8.1, 7.6, 7.0, 7.2, 8.1 and 8.5 us with 1, 2, 3, 4, 5, 6 and 8; 1024 x 17408: 40.4, 24.7, 18.8, 15.5, 14.2, 14.1 and 13.1.  Pairs, 256 rows,
// 5120 x 17408: 59.5, 48.0 and 38.2 with 1, 2 and 3, and single blocks, which cannot be split there, 54.0; 5120 x 5120: 18.6, 21.8 and 20.0, and 15.6.)
template <int CW>
constexpr int kExchange = paired(CW) ? 1200 : 330;  // 10 ns
template <int CW>
constexpr int kMaxSplit = paired(CW) ? 3 : kMaxCluster;  // (four pairs gain from 290 blocks of columns on)
template <int CW>
int split_of(long long tiles, int n_k) {
    constexpr int kEach = paired(CW) ? 55 : 27;  // 10 ns
    int best = 1, least = n_k * kEach;
    for (int split = 2; split <= (kMaxSplit<CW>) && n_k >= 2 * split; ++split) {
        const int fit = Variant<CW, true>::clusters(split), takes = n_k * kEach / split + kExchange<CW> + (2 * tiles > fit ? 220 : 3 * tiles > fit ? 80 : 0);
        if (tiles <= fit && (!turned(CW) || takes <= least)) best = split, least = takes;
    }
    return best;
}

template <int CW>
cudaError_t launch(QmmF8 a, const QmmF8Args &in, cudaStream_t stream) {
    using One = Variant<CW, false>;
    constexpr bool PAIR = paired(CW), TURNED = turned(CW);
    constexpr int kStage = kABytes + (TURNED ? kRows : 2 * CW) * kQCols, kTile = One::kGroup * kRows;
    a.tok_tiles = TURNED ? (in.ntok + kTile - 1) / kTile : 1;
    a.row_tiles = (in.rows + kTile - 1) / kTile;
    a.half_sm = One::kHalf;
    a.b_bytes = kStage - kABytes;
    const long long tiles = static_cast<long long>(a.row_tiles) * a.tok_tiles;
    if (tiles > (1ll << 30)) return cudaErrorInvalidValue;
    a.split = split_of<CW>(tiles, a.n_k);
    const bool brief = a.n_k <= 8 * a.split;  // a few stages for each block: what counts is how soon it begins and ends
    // Sums have memory of their own where that costs no stage or the stages are few, else they go where the stages were, one barrier of the cluster later.
    const int room = a.split > 1 ? CW / 8 * ((kWriters + a.split - 1) / a.split) * (a.split - 1) * 1024 : 0;
    const int whole = a.split > 1 ? One::kSmem - 1024 : One::kRoom, beside = (whole - room) / kStage;  // (what is split has no outputs on their way)
    a.stages = whole / kStage;
    if (a.split > 1 && (beside == a.stages || (brief && beside >= 3))) a.exchange = whole - room, a.stages = beside;
    if (a.stages > kMaxStages) a.stages = kMaxStages;
    Maps<TURNED> maps{};
    cudaError_t err = encode_rows(&maps.w, in.w, in.cols, in.w_pitch, in.rows, PAIR ? kRows / 2 : kRows);
    if (err == cudaSuccess) err = encode_rows(&maps.q, in.q, in.cols, f8_pitch(in.cols), in.ntok, TURNED ? kRows : 2 * CW);
    if constexpr (TURNED) {
        a.tile_out = a.split == 1 && !in.add && static_cast<long long>(in.rows) * in.y_elem % 16 == 0;
        if (a.tile_out && err == cudaSuccess) err = encode_outputs(&maps.y, in.y, in.rows, in.ntok, in.y_elem);
    }
    if (err != cudaSuccess) return err;
    if (a.split > 1) return Variant<CW, true>::launch(maps, a, in.overlap, stream);
    return One::launch(maps, a, in.overlap, stream);
}

// What blocks (pairs) of all tiles take, in 10 ns: a pair 0.55 us for a block of columns of 256 x 256 outputs, a single block 0.39 for 128 x 128, where all have work.
template <int CW>
long long takes(int rows, int ntok, int n_k) {
    constexpr int kTile = Variant<CW, false>::kGroup * kRows, kEach = paired(CW) ? 55 : 39;
    const long long tiles = static_cast<long long>((rows + kTile - 1) / kTile) * ((ntok + kTile - 1) / kTile);
    const int fit = Variant<CW, false>::clusters(1), split = split_of<CW>(tiles, n_k);
    if (fit == 0) return LLONG_MAX;
    return split > 1 ? n_k * kEach / split + kExchange<CW> : (tiles + fit - 1) / fit * n_k * kEach;
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
    // (6144 x 5120 with 256 rows: pairs 30.9 us, single blocks 15.9; with 512 21.6 and 27.1)
    if (in.ntok > 128 && takes<128>(in.rows, in.ntok, a.n_k) < takes<64>(in.rows, in.ntok, a.n_k)) return launch<128>(a, in, stream);
    if (in.ntok > 64) return launch<64>(a, in, stream);
    if (in.ntok > 32) return launch<32>(a, in, stream);
    return in.ntok > 16 ? launch<16>(a, in, stream) : launch<8>(a, in, stream);
}

}  // namespace vqm
