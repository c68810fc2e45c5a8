// q3s_attn_maps.cuh -- host side: the tensor maps of the attention kernels.
#pragma once

#include <cuda.h>

#include <algorithm>
#include <cstdint>

#include "q3s_attn.cuh"
#include "q3s_tma.cuh"

namespace q3s {

// Tensor maps: q as [T, q_heads, dim] in boxes of a tile's tokens by a group's
// heads by 64 dims; a cache as [blocks, kv_heads, dim / 64, block_size, 64]
// (the dims cut into slices of the swizzle's 128 bytes) in boxes of `slices`
// slices of one page, at most `tokens` of it; zeros outside.  An axis of one
// entry has no stride of its own: any that the encoder takes.
inline bool encode(CUtensorMap* m, bool bf16, const void* base, int rank, const int64_t* dims, const int64_t* strides,
            const int* box) {
  const EncodeTiled enc = encode_tiled();
  if (!enc) return false;
  cuuint64_t d[5], s[4];
  cuuint32_t b[5], ones[5] = {1, 1, 1, 1, 1};
  for (int i = 0; i < rank; ++i) {
    d[i] = static_cast<cuuint64_t>(dims[i]);
    b[i] = static_cast<cuuint32_t>(box[i]);
    if (i) s[i - 1] = static_cast<cuuint64_t>(2 * (dims[i] > 1 ? strides[i - 1] : 64));
  }
  return enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank,
             const_cast<void*>(base), d, s, b, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
inline bool query_map(const AttnArgs& a, int dim, bool bf16, int per_tile, CUtensorMap* q) {
  const int64_t dims[3] = {dim, a.Hq, a.T}, strides[2] = {a.qh, a.qt};
  const int box[3] = {64, a.G, per_tile};
  return encode(q, bf16, a.q, 3, dims, strides, box);
}
inline bool cache_maps(const AttnArgs& a, int dim, bool bf16, int tokens, int slices, CUtensorMap* k, CUtensorMap* v) {
  const int64_t dims[5] = {64, a.bs, dim / 64, a.H, a.blocks};
  const int64_t ks[4] = {a.kp, 64, a.kh, a.kb}, vs[4] = {a.vp, 64, a.vh, a.vb};
  const int box[5] = {64, std::min(a.bs, tokens), slices, 1, 1};
  return encode(k, bf16, a.k, 5, dims, ks, box) && encode(v, bf16, a.v, 5, dims, vs, box);
}

}  // namespace q3s
