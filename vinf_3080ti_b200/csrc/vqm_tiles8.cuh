// What the products of 8-bit rows (vqm_qmm_i8.cu, vqm_qmm_f8.cu) have in common: tiles of 128 columns that come by TMA into a ring of stages and are
// multiplied by tcgen05.mma, bounded waits, pairs and clusters of blocks.
#pragma once

#include <cuda.h>

#include "vqm_kernels.h"
#include "vqm_tcmv.cuh"

namespace vqm {
namespace {

constexpr int kQCols = 128;  // columns of a stage

using tc::bar_arrive, tc::bar_init, tc::bar_try, tc::bar_try_cluster, tc::in_block, tc::s32;

// A test has one part of a tile's columns multiply no more than the first block of them, so that waits run out.
#ifdef VQM_STALLED_PART
__device__ __forceinline__ bool stalled(int part, int done) { return part == VQM_STALLED_PART && done >= 1; }
#else
__device__ __forceinline__ constexpr bool stalled(int, int) { return false; }
#endif

// Bounded; false once this or another wait of the block has given up.  A wait that succeeds looks at nothing but its barrier: the loops below have some
// 500 cycles per stage.
template <bool CLUSTER>
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int *failed) {
    unsigned long long began = 0;
#pragma unroll 1
    for (uint32_t i = 1;; ++i) {
        if (CLUSTER ? bar_try_cluster(bar, parity) : bar_try(bar, parity)) return true;
        if ((i & 255u) == 0 && tc::give_up(&began, failed)) return false;
    }
}

__device__ __forceinline__ uint64_t tile_desc(uint32_t addr) {  // K-major, 128-byte swizzle, groups of 8 rows 1024 bytes apart
    return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (1ull << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void copy_tile(uint32_t to, const CUtensorMap *map, int x, int row, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(to), "l"(map), "r"(x), "r"(row), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Arrives on the barrier (in both blocks of pair `pair`) once the MMAs issued so far are done.
template <bool PAIR>
__device__ __forceinline__ void commit(uint32_t bar, uint32_t pair) {
    if constexpr (PAIR) {
        const uint16_t both = static_cast<uint16_t>(3u << (2 * pair));
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"(both) : "memory");
    } else {
        tc::commit(bar);
    }
}

// 8-bit rows as a 2-D tensor; a tile is 128 columns of `box_rows` rows.  Columns and rows beyond the last arrive as zeros.
inline cudaError_t encode_rows(CUtensorMap *map, const void *rows_at, int cols, long long pitch, int rows, int box_rows) {
    TcEncode encode = nullptr;
    if (const cudaError_t err = tc_encoder(&encode); err != cudaSuccess) return err;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)}, strides[1] = {static_cast<cuuint64_t>(pitch)};
    const cuuint32_t box[2] = {kQCols, static_cast<cuuint32_t>(box_rows)}, elem[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(rows_at), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? cudaSuccess
               : cudaErrorInvalidValue;
}

}  // namespace
}  // namespace vqm
