// Tensor maps of the paged cache and of packed rows, and the TMA loads of their boxes:
// what the attention kernels of runs share. A box lands as groups of eight tokens,
// [group][block of 64 dims][token of the group][64 dims] with the 128-byte swizzle.
#pragma once

#include "chunk_common.cuh"
#include "umma_common.cuh"

namespace b200kv {

constexpr int kBoxDims = 256;

// One box of a page: `box` tokens x kBoxDims, token groups of eight from `token_group`.
__device__ __forceinline__ void tma_load_page_box(uint32_t dst, const CUtensorMap *map, int block,
                                                  int token_group, int head, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(0), "r"(block), "r"(token_group),
      "r"(head), "r"(bar)
      : "memory");
}
// Eight packed rows x kBoxDims; rows past the tensor arrive as zeros.
__device__ __forceinline__ void tma_load_rows_box(uint32_t dst, const CUtensorMap *map, int block,
                                                  int row, int head, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(row), "r"(block), "r"(head), "r"(bar)
      : "memory");
}

// Tokens per box: the largest power of two up to `most` that divides the page (a box
// then lies in one page); less than eight rows do not fill a swizzle atom (0).
inline int box_tokens(int page_size, int most) {
  int box = most;
  while (page_size % box != 0) box /= 2;
  return box >= 8 ? box : 0;
}

inline bool make_cache_map(CUtensorMap *map, const __nv_bfloat16 *base, const Gemma4KvCacheConfig &c, int box) {
  EncodeTiledFn encode = encode_tiled_fn();
  if (encode == nullptr) return false;
  const cuuint64_t row = cuuint64_t(c.num_heads) * c.head_dim * 2;
  // [head][group of 8 tokens][block of 64 dims][token of the group][64 dims]: the
  // pages of all layers are one row of tokens, of which a box takes whole groups
  const cuuint64_t dims[5] = {64, 8, cuuint64_t(c.head_dim / 64),
                              cuuint64_t(c.num_layers) * c.num_pages * (c.page_size / 8),
                              cuuint64_t(c.num_heads)};
  const cuuint64_t strides[4] = {row, 128, row * 8, cuuint64_t(c.head_dim) * 2};
  const cuuint32_t boxes[5] = {64, 8, kBoxDims / 64, cuuint32_t(box / 8), 1};
  const cuuint32_t steps[5] = {1, 1, 1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<__nv_bfloat16 *>(base), dims,
                strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

inline bool make_rows_map(CUtensorMap *map, const __nv_bfloat16 *base, int rows, int heads, int head_dim) {
  EncodeTiledFn encode = encode_tiled_fn();
  if (encode == nullptr) return false;
  const cuuint64_t row = cuuint64_t(heads) * head_dim * 2;
  const cuuint64_t dims[4] = {64, cuuint64_t(rows), cuuint64_t(head_dim / 64), cuuint64_t(heads)};
  const cuuint64_t strides[3] = {row, 128, cuuint64_t(head_dim) * 2};
  const cuuint32_t box[4] = {64, 8, kBoxDims / 64, 1};
  const cuuint32_t steps[4] = {1, 1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<__nv_bfloat16 *>(base), dims,
                strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace b200kv
