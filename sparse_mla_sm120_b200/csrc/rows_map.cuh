// Tensor maps: the one by which TMA gathers packed 656-byte rows, and their making.
#pragma once

#include <cuda.h>

#include "common.cuh"

namespace smla {

constexpr int NO_ROW = 0x7fffffff;             // outside the tensor map: arrives as zeros

// One cache whose rows lie one after the other (pages without padding between them), on a 16-byte boundary: what a tensor map
// needs to name them by their index.
inline bool one_linear_array(const AttnParams& p) {
    return p.layout == SMLA_LAYOUT_V32 && p.extra_topk == 0 && p.block_stride == (int64_t)p.page_block_size * ROW_BYTES &&
           (reinterpret_cast<uintptr_t>(p.kv) & 15u) == 0;
}

// A map of `rank` dimensions with 128B swizzle: strides in bytes, of all dimensions but the first.  0 or an error code.
int encode_map(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base, const uint64_t* dims, const uint64_t* strides, const uint32_t* box,
               CUtensorMapL2promotion promotion);

// The cache as 32-bit words, 164 per row; boxes of 32 words (128 bytes) of one row, 128B swizzle.  0 or an error code.
int rows_tensor_map(const uint8_t* kv, CUtensorMap* map);
// paged_pair.cu
int launch_attn_paged_pair(const PagedParams& p, bool f16, const CUtensorMap& q_map, const CUtensorMap& k_map, cudaStream_t stream);

}  // namespace smla
