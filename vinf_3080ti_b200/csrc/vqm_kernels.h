// Host-visible declarations shared by the kernel translation units and the runtime.
#pragma once

#include <cuda.h>  // CUtensorMap (types only; nothing links against the driver)
#include <cuda_runtime.h>

#include <cstdint>

namespace vqm {

// Memory that a call reads or writes; none: at a null pointer.
struct Extent {
    const void *at;
    size_t bytes;
};
constexpr Extent kNoExtent{nullptr, 0};
inline bool overlap(const Extent &a, const Extent &b) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(a.at), q = reinterpret_cast<uintptr_t>(b.at);
    return a.at != nullptr && b.at != nullptr && (p <= q ? q - p < a.bytes && b.bytes > 0 : p - q < b.bytes && a.bytes > 0);
}

// Attributes of a launch, of which `attr` holds two; returns how many there are.  overlap: programmatic stream serialization, with which the blocks
// may begin while the kernel before them in the stream still runs (they wait for its end themselves, but for weights, which are in place).
// cluster: blocks of a cluster, 0 for none.
inline unsigned launch_attributes(cudaLaunchAttribute *attr, bool overlap, int cluster) {
    unsigned n = 0;
    if (overlap) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    if (cluster > 0) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = static_cast<unsigned>(cluster);
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    return n;
}

constexpr int kMaxParts = 4;  // tensors one launch can cover (they share the activations, the type and the columns)

// Row-sharded matvec across GPUs: where a launch stores its outputs inside every rank's exchange region (plain remote
// stores over NVLink, issued by the lane that holds the output) and which flags order that against the consumers.
struct PushInfo {
    unsigned long long region[8];  // device address of every rank's exchange region, this rank's included
    unsigned *pushes;              // this rank's own count of pushes per slot, unsigned[n_slots] (inside its region)
    long long dst_off[kMaxParts];  // per tensor: byte offset, inside a region, of its gathered y[0][0]
    long long flag_off;            // byte offset, inside a region, of the flag table: unsigned flags[slot][8 ranks], the
                                   // number of pushes of the slot each rank has completed
    int n_ranks, rank;
    int rows_total[kMaxParts];     // per tensor: the gathered tensor has rows_total rows ...
    int row_begin[kMaxParts];      // ... and this rank's slice starts at row_begin
    int push_slot;                 // 1 + flag slot signalled after the push (0: no push)
    int wait_slot;                 // 1 + slot every rank must have pushed as often as this rank before x is read (0: no wait)
};

// One tensor of a launch.  The launch numbers the rows of its tensors consecutively; tensor p owns launch rows
// [row_end of tensor p - 1, row_end).  Unused entries have row_end = INT_MAX.
struct MatvecPart {
    const uint8_t *w;  // raw blocks, readable up to 15 bytes past the end
    float *y;          // [M][rows] fp32 (may be null when only the argmax is wanted)
    int row_end;
    int rows;          // rows of this tensor (the stride of y)
};

struct MatvecArgs {
    MatvecPart part[kMaxParts];
    const float *x;          // [M][cols] fp32, 16-byte aligned
    const uint8_t *codebook;  // device copy of the type's GGUF codebook (IQ2/IQ3 types), else null
    unsigned *status;        // device error word (0 = fine)
    // fused argmax (all null / 0 when unused; single-tensor launches only)
    float *part_val;         // [kMaxTok][gridDim.x]
    int *part_idx;           // [kMaxTok][gridDim.x]
    unsigned *done_counter;  // zero before the launch; the kernel leaves it zero
    int *out_idx;            // [M] winning row (+ row_base), 0x7fffffff if the column has no value above -inf
    float *out_val;          // [M] winning value (may be null)
    int rows, cols;          // rows: of all tensors together
    long long row_bytes;
    int row_base;            // added to row numbers reported by the argmax (row-sharded weights)
    // Column split for short launches: the k_split blocks of a thread-block cluster share a group of rows (one row per
    // warp), each takes a range of the column segments and leaves its partial sums in the shared memory of the
    // cluster's first block, which adds them in the order of k and writes the outputs.
    int k_split;             // chosen by the launcher (from the rows and the columns only, never from M); 1 = off
    int allow_split;         // host only: the caller permits the split
    int overlap_launch;      // host only: launch with programmatic stream serialization (see qmv_kernel)
    int max_grid;            // host only: upper bound on the grid (0 = none); sizes the argmax partial arrays
    // Fused prologue / epilogue (the flags of the reference's megakernel QMV, engine/csrc/common/qwen_mk_abi.h:55-58):
    //   kFuseSiluMul: the activations are silu(x) * x2;  kFuseNorm: then rmsnorm over the columns times norm_w;
    //   kFuseAdd: y += W x instead of y = W x (the outputs already hold the residual).
    int fuse;                // kFuse* bits, 0 = plain matvec
    const float *x2;         // [M][cols], with kFuseSiluMul
    const float *norm_w;     // [cols], with kFuseNorm
    float eps;               // rmsnorm epsilon
    PushInfo push;           // all zero when the tensor is not sharded
};

// What the tensor-core matvec needs beside that; filled in by its launcher, so that no block starts with integer divisions.  (Not
// in MatvecArgs: with these 64 bytes the CUDA-core kernel's small launches take 1 to 3 % longer, 3.07 instead of 2.98 us.)
static_assert(sizeof(MatvecArgs) <= 384, "parameters of the CUDA-core kernel");
struct TcMatvecArgs : MatvecArgs {
    const uint8_t *x_split;  // ready-made B operands of more than 8 activation rows
    float *partials;         // sums of launches whose columns are split, see tc_finish_tile; null: clusters exchange them
    unsigned *partial_counts;  // [tile]: how many column ranges are there; zero before and after a launch
    int tc_groups, tc_split_recip;  // groups of k_split blocks, and 65536 / k_split rounded up
    int tc_steps[9];         // block k of a group takes the 256-column steps [tc_steps[k], tc_steps[k + 1])
    int tc_deal, tc_deal_recip;  // rows of a tile that each block of a cluster finishes, and 65536 / tc_deal rounded up
    int tc_first, tc_end;        // tiles of this launch (a launch may take the last round of another, see choose_tc_tail)
    unsigned char tc_map_shift[kMaxParts];  // log2 of the number of tensor maps of each tensor
};

enum : int { kFuseAdd = 1, kFuseNorm = 2, kFuseSiluMul = 8 };  // (4 is the fused argmax, which has its own fields)

constexpr int kMaxSplit = 8;  // column ranges a row can be split into (the portable cluster size)

enum : unsigned { kStatusOk = 0, kStatusWaitExpired = 1, kStatusPeerWaitExpired = 2 };

// One launcher per GGUF type (vqm_matvec_type.cu).  m: activation rows (1..8); sm_count: SMs of the device;
// grid_out (optional) receives the grid size used.
#define VQM_FOR_EACH_TYPE(X) \
    X(0, F32) X(1, F16) X(8, Q8_0) X(10, Q2_K) X(11, Q3_K) X(12, Q4_K) X(13, Q5_K) X(14, Q6_K) X(16, IQ2_XXS) \
    X(17, IQ2_XS) X(18, IQ3_XXS) X(20, IQ4_NL) X(21, IQ3_S) X(22, IQ2_S) X(23, IQ4_XS)
#define VQM_DECLARE_LAUNCHER(id, name)                                                                            \
    cudaError_t launch_qmv_##name(const MatvecArgs &a, int m, int sm_count, cudaStream_t stream, int *grid_out); \
    cudaError_t launch_qmv_fused_##name(const MatvecArgs &a, int m, int sm_count, cudaStream_t stream, int *grid_out);  // honours a.fuse
VQM_FOR_EACH_TYPE(VQM_DECLARE_LAUNCHER)
#undef VQM_DECLARE_LAUNCHER

constexpr int kTcTileRows = 256;   // rows of a tile of the tensor-core matvec
constexpr int kTcMaxMagnitude = 66;  // of a codebook, for the tensor-core matvec: times 31 it has to fit into the 11 bits of fp16
inline int tc_tiles(const MatvecArgs &a) {
    int n = 0;
    for (int p = 0; p < kMaxParts; ++p) n += (a.part[p].rows + kTcTileRows - 1) / kTcTileRows;
    return n;
}
// Room for the partial sums of a launch whose columns are split.  It holds a record of every block of one that takes each tile at once (not where
// blocks take several tiles): at most sm_count / 2 tiles, sm_count blocks.  The counts, then the records of tc_finish_tile, 2 of a block for up to 8 activation rows, 12 smaller ones for 24.
constexpr bool tc_partials_hold(int n_tiles, int k_split, int sm_count) { return static_cast<long long>(n_tiles) * k_split <= sm_count; }
constexpr size_t tc_partial_count_bytes(int sm_count) { return (static_cast<size_t>(sm_count) * 4 + 255) / 256 * 256; }
constexpr size_t tc_partial_bytes(int sm_count, int m) {
    return tc_partial_count_bytes(sm_count) + static_cast<size_t>(sm_count) * (m <= 8 ? 2 * (4 * kTcTileRows + 32) : 12 * (2 * kTcTileRows + 32)) * 4;
}
constexpr size_t kTcPartialAlign = 256;  // of the room's address; the kernels' accesses to it are of up to 16 bytes
// Size of the scratch for the B operands of more than 8 activation rows that is to hold `need` bytes where `present` do not: a multiple of
// kTcPartialAlign, because room for partial sums lies behind it.  At most 42 KB per 256 columns; 4 MB hold 24576 columns of any type, so that a
// runtime allocates once (with 3.9 MB for partial sums behind them).  (cudaMalloc takes 330 us for any size from 1 to 16 MB; with 2 MB, which
// tensors of more than 12288 columns outgrow, to bind three tensors and their buffers of 24 rows took 1720 us instead of 1480.)  It grows by half
// at least: what it has outgrown, which captured graphs may use, is together at most twice its size.
constexpr size_t tc_grown_split_bytes(size_t need, size_t present) {
    size_t bytes = need < (4u << 20) ? 4u << 20 : need;
    if (bytes < present + present / 2) bytes = present + present / 2;
    return (bytes + kTcPartialAlign - 1) / kTcPartialAlign * kTcPartialAlign;
}
struct TcScratch {
    const uint8_t *x_split = nullptr;  // the B operands of more than 8 activation rows
    // Room for partial sums, aligned to kTcPartialAlign, in use by one launch at a time: counts zero and sums empty (bytes of 0xFF) before and
    // after it.  Null: the blocks that share columns are clusters and exchange sums in shared memory.  The outputs are the same, bit for bit.
    uint8_t *partials = nullptr;
};
// The tensor-core matvec (vqm_tcmv_type.cu).  maps: per tensor of the launch its tensor maps (tc_encode_maps).
#define VQM_FOR_EACH_TC_TYPE(X) \
    X(8, Q8_0) X(10, Q2_K) X(11, Q3_K) X(12, Q4_K) X(13, Q5_K) X(14, Q6_K) X(16, IQ2_XXS) X(17, IQ2_XS) X(18, IQ3_XXS) \
    X(20, IQ4_NL) X(21, IQ3_S) X(22, IQ2_S) X(23, IQ4_XS)
// split_tcmv_*: into how many column ranges the launch would be split (to go into a.k_split), 0 = the CUDA-core kernel is better.
// launch_tcmv_*: n_launched (may be null) is counted up by the kernels launched, one or two (split: one for 16 rows).
#define VQM_DECLARE_TC_LAUNCHER(id, name)                                                                                        \
    int split_tcmv_##name(const MatvecArgs &a, int sm_count);                                                                    \
    cudaError_t launch_tcmv_##name(const MatvecArgs &a, const CUtensorMap *const *maps, int n_parts, const TcScratch &scratch, int m, \
                                   int sm_count, cudaStream_t stream, int *n_launched);
// wide_rows_*: how many activation rows a launch takes, 24, 16 or 8; split_bytes_*: size of x_split for a launch of more than 8 rows over so
// many columns, 0 if the type takes 8 at most; launch_split_*: makes it from a.x.
#define VQM_DECLARE_SPLIT(id, name)                   \
    int wide_rows_##name();                            \
    size_t split_bytes_##name(int cols);               \
    cudaError_t launch_split_##name(const MatvecArgs &a, uint8_t *x_split, int m, cudaStream_t stream, int *n_launched);
VQM_FOR_EACH_TC_TYPE(VQM_DECLARE_SPLIT)
#undef VQM_DECLARE_SPLIT
VQM_FOR_EACH_TC_TYPE(VQM_DECLARE_TC_LAUNCHER)
#undef VQM_DECLARE_TC_LAUNCHER
// box_rows: rows of a class that one copy brings (32: a tile of 256 rows in all)
cudaError_t tc_encode_maps(int type, const uint8_t *w, int rows, long long row_bytes, int box_rows, CUtensorMap *out);

constexpr int kMaxGrid = 4096;  // upper bound on the matvec grid (sizes the argmax partial arrays)

// Prompt-pass GEMM on the tensor cores (vqm_gemm.cu).  xh: fp16 activations [ntok padded to gemm_token_tile()][cols].
int gemm_token_tile();
// overlap: see launch_attributes
cudaError_t launch_f32_to_f16_rows(const float *x, void *xh, long long n_valid, long long n_total, bool overlap, cudaStream_t stream);
cudaError_t launch_qgemm(int type, const uint8_t *w, const void *xh, float *y, int rows, int cols, long long row_bytes, int ntok,
                         const uint8_t *codebook, cudaStream_t stream);

// Prompt-pass GEMM on tcgen05 tensor cores with the accumulators in tensor memory (vqm_gemm_tc5.cu); xh: ntok rows, needs
// cols to be a multiple of 64.  status: device word that receives a code if a bounded
// wait expires.
bool gemm_tc5_supports(int cols);
cudaError_t launch_qgemm_tc5(int type, const uint8_t *w, const void *xh, float *y, int rows, int cols, long long row_bytes, int ntok,
                             const uint8_t *codebook, unsigned *status, bool overlap, cudaStream_t stream);

// n16 16-byte words from pinned host memory
cudaError_t launch_fetch(const void *from, void *to, int n16, cudaStream_t stream);

// ---- 8-bit integer passes (vqm_rows_i8.cu, vqm_qmm_i8.cu) and the verification of drafted tokens (vqm_verify.cu) ----

constexpr int kI8Rows = 24;          // type id of a weight tensor of 8-bit integer rows with a scale each (VQM_I8_ROWS)
constexpr int kI8MaxCols = 131071;   // (2^17 - 1) * 2^14 still fits into a 32-bit sum
constexpr int kI8MaxRows = 1 << 30;  // (sums of a row and a tile fit into 32 bits)
__host__ __device__ constexpr long long i8_pitch(int cols) { return (static_cast<long long>(cols) + 15) / 16 * 16; }  // bytes from one row of 8-bit values to the next

struct RowsI8Args {
    const void *x;         // [ntok][cols] of `elem` bytes
    const void *x2;        // the values are silu(x) * x2; or null
    const void *residual;  // the values are x + residual, and go to `total` as well (which may be either of them); or null
    void *total;
    const float *norm_w;   // rmsnorm over the columns times these; or null
    int8_t *q;             // [ntok][i8_pitch(cols)], zeros behind the last column
    float *scales;         // [ntok]
    int cols, ntok, elem;
    float eps;
    double inv_cols;       // 1 / cols, filled in by the launcher
};
// overlap: see launch_attributes
cudaError_t launch_rows_i8(const RowsI8Args &a, bool overlap, int sm_count, cudaStream_t stream);
// How far fp32 leaves t = n / s from its value, relative to t: whoever is that near to a half is rounded in 64 bits.  In units of 2^-24: the product with the
// norm's weights 1, its factor r 1, the division of r by s 1, the product with that 1, and the rounding of the bound itself, half a unit at |t| = 1/2.
// Gated values have two products before the division instead, and the sigmoid: 4 of ex2, 1 of the sum, 2 of the reciprocal, and for each unit of -x (largest
// of the thread) 1 of the argument and 0.23 of the constant in it.
constexpr float kI8Off = 5.0f / (1 << 24), kI8GatedOff = 12.0f / (1 << 24), kI8GatedOffPerX = 1.35f / (1 << 24);

struct QmmI8Args {
    const int8_t *w;       // [rows][w_pitch], 16-byte aligned, w_pitch a multiple of 16
    const float *w_scales;
    const int8_t *q;       // [ntok][i8_pitch(cols)]
    const float *q_scales;
    void *y;               // [ntok][rows] of y_elem bytes
    long long w_pitch;
    int rows, cols, ntok, y_elem;
    bool add;              // y += instead of y =
    bool overlap;          // see launch_attributes
    unsigned *status;      // device word that receives a code if a bounded wait expires
};
cudaError_t launch_qmm_i8(const QmmI8Args &a, cudaStream_t stream);

struct VerifyArgs {
    const void *target;        // [seqs][drafts + 1][vocab] of `elem` bytes
    const void *draft;         // [seqs][drafts][vocab], or null: the drafts have no probabilities of their own
    const int *tokens;         // [seqs][drafts]
    const int *lens;           // [seqs] drafts of each sequence; or null: all
    const float *uniforms;     // [seqs][drafts + 1]
    const float *temperature;  // [seqs]; or null: 1
    int *out;                  // [seqs][drafts + 2]; all -1 if the status word is not 0
    const unsigned *status;    // device word with the code of a wait that has expired: the logits may not be what they should
    int vocab, seqs, drafts, elem;
};
// overlap: see launch_attributes
cudaError_t launch_verify(const VerifyArgs &a, bool overlap, cudaStream_t stream);
// How far from one another, relative to the larger, the two sides of a draft's test may be if they are equal but come from fp32 sums of exponentials, of
// which a lane adds up `adds` parts.  In units of 2^-24: a part is added with one rounding, and where it has a new largest the sum before it is scaled, 4 of
// ex2 and 1 of the product; both sides have such a sum, and the products of so many factors add less than 5 %.  The rest is 2e-5: 4 of each ex2, 3 times
// its argument (over a row at most the logarithm of its length, 22, on average), 10 of the additions within a part, 90 of 15 joins of lanes, warps and blocks.
// Beyond 32768 parts (16.7 million logits to a block) nothing is taken for sure.
__host__ __device__ constexpr double verify_band(long long adds) { return adds > 32768 ? 2.0 : 1e-4 + 1.05 * 12.0 / (1 << 24) * static_cast<double>(adds); }

// ---- Passes in 8-bit floating point (vqm_rows_f8.cu, vqm_qmm_f8.cu) and log probabilities (vqm_logprobs.cu) ----

constexpr int kF8Blocks = 128;       // type id of a weight tensor of e4m3 values with a scale for each block of 128 x 128 (VQM_F8_BLOCKS)
constexpr int kF8Block = 128;        // columns (and weight rows) that share a scale
constexpr int kF8MaxCols = 1 << 20;
constexpr int kF8MaxRows = 1 << 30;
__host__ __device__ constexpr long long f8_pitch(int cols) { return (static_cast<long long>(cols) + 15) / 16 * 16; }  // bytes from one row of 8-bit values to the next
__host__ __device__ constexpr int f8_blocks(int n) { return (n + kF8Block - 1) / kF8Block; }
__host__ __device__ constexpr long long f8_scale_pitch(int ntok) { return (static_cast<long long>(ntok) + 3) / 4 * 4; }  // floats from the scales of one block of columns to those of the next

struct RowsF8Args {
    const void *x;         // [ntok][cols] of `elem` bytes
    const void *x2;        // the values are silu(x) * x2; or null
    const void *residual;  // the values are x + residual, and go to `total` as well (which may be either of them); or null
    void *total;
    const float *norm_w;   // rmsnorm over the columns times these; or null
    uint8_t *q;            // [ntok][f8_pitch(cols)], zeros behind the last column
    float *scales;         // [f8_blocks(cols)][f8_scale_pitch(ntok)]
    int cols, ntok, elem;
    float eps;
};
// overlap: see launch_attributes
cudaError_t launch_rows_f8(const RowsF8Args &a, bool overlap, int sm_count, cudaStream_t stream);
// e4m3 blocks of 128 x 128 and their scales from fp32 rows: w [rows][cols] -> q [rows][f8_pitch(cols)], scales [f8_blocks(rows)][f8_blocks(cols)]
cudaError_t launch_blocks_f8(const float *w, uint8_t *q, float *scales, int rows, int cols, cudaStream_t stream);

struct QmmF8Args {
    const uint8_t *w;      // [rows][w_pitch], 16-byte aligned, w_pitch a multiple of 16
    const float *w_scales; // [f8_blocks(rows)][f8_blocks(cols)]
    const uint8_t *q;      // [ntok][f8_pitch(cols)]
    const float *q_scales; // [f8_blocks(cols)][f8_scale_pitch(ntok)]
    void *y;               // [ntok][rows] of y_elem bytes
    long long w_pitch;
    int rows, cols, ntok, y_elem;
    bool add;              // y += instead of y =
    bool overlap;          // see launch_attributes
    unsigned *status;      // device word that receives a code if a bounded wait expires
};
cudaError_t launch_qmm_f8(const QmmF8Args &a, cudaStream_t stream);

constexpr int kMaxTop = 32;  // alternatives of a row (VQM_MAX_TOP)
struct LogprobsArgs {
    const void *logits;        // [rows][vocab] of `elem` bytes
    const int *tokens;         // [rows]
    const float *temperature;  // [rows]; or null: 1
    float *out, *entropy;      // [rows]; entropy may be null
    int *top_ids;              // [rows][top]
    float *top_out;            // [rows][top]; or null
    const unsigned *status;    // device word with the code of a wait that has expired: the logits may not be what they should
    int vocab, rows, top, elem;
};
// overlap: see launch_attributes
cudaError_t launch_logprobs(const LogprobsArgs &a, bool overlap, cudaStream_t stream);

cudaError_t launch_argmax_rows(const float *x, int n, int ntok, int *out, cudaStream_t stream);
cudaError_t launch_dequant(int type, const uint8_t *w, float *out, long long numel, const uint8_t *codebook,
                           cudaStream_t stream);

}  // namespace vqm
