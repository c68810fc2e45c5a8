// q3s_chunk.cu -- host side of q3s_chunk_attention.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "q3s_attn_maps.cuh"
#include "q3s_chunk.cuh"
#include "q3s_tma.cuh"

namespace {

struct Layout {
  int64_t cuts, part_ml, part_o, bytes;  // byte offsets
  int per_tile, slot_rows, ctas;
};

Layout layout_of(const q3s_chunk_attention_desc* d) {
  Layout l;
  const int G = d->q_heads / d->kv_heads;
  l.per_tile = q3s::CH_M / G;
  l.slot_rows = std::min(2 * l.per_tile, std::max(d->tokens, 1)) * G;
  l.ctas = q3s::sm_count();
  auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
  const int64_t rows = static_cast<int64_t>(2) * l.ctas * l.slot_rows;
  l.cuts = 0;
  l.part_ml = up(static_cast<int64_t>(l.ctas) * sizeof(q3s::ChunkCut));
  l.part_o = l.part_ml + up(rows * 8);
  l.bytes = l.part_o + up(rows * d->dim * 4);
  return l;
}

q3s_status check_sizes(const q3s_chunk_attention_desc* d) {
  using q3s::report;
  if (!d) return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_chunk_attention: desc is NULL");
  if (d->struct_size != sizeof(q3s_chunk_attention_desc))
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_chunk_attention: struct_size %u != %u (ABI mismatch)", d->struct_size,
                  static_cast<unsigned>(sizeof(q3s_chunk_attention_desc)));
  if (d->batch < 0 || d->batch > Q3S_MAX_CACHE_ROWS || d->tokens < 0)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_chunk_attention: batch %d is not in [0, %d] or tokens %d is negative", d->batch,
                  Q3S_MAX_CACHE_ROWS, d->tokens);
  if (d->kv_heads < 1 || d->q_heads < 1 || d->q_heads % d->kv_heads || d->q_heads / d->kv_heads > Q3S_MAX_CHUNK_GROUP)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_chunk_attention: %d query heads are not 1 to %d for each of %d key/value heads",
                  d->q_heads, Q3S_MAX_CHUNK_GROUP, d->kv_heads);
  if (d->kv_heads > 65535)
    return report(Q3S_ERR_UNSUPPORTED, "q3s_chunk_attention: %d key/value heads are too many", d->kv_heads);
  if (d->dim != 64 && d->dim != 128)
    return report(Q3S_ERR_UNSUPPORTED, "q3s_chunk_attention: dim %d is not 64 or 128", d->dim);
  if (d->block_size != 16 && d->block_size != 32 && d->block_size != 64 && d->block_size != 128)
    return report(Q3S_ERR_UNSUPPORTED, "q3s_chunk_attention: block_size %d is not 16, 32, 64 or 128", d->block_size);
  if (d->elem != Q3S_ELEM_BF16 && d->elem != Q3S_ELEM_F16)
    return report(Q3S_ERR_UNSUPPORTED, "q3s_chunk_attention: elem %d is not bf16 or f16", d->elem);
  if (d->blocks < 1 || d->max_blocks < 0 || d->prefix_length < 0 || d->window < 0)
    return report(Q3S_ERR_INVALID_ARGUMENT,
                  "q3s_chunk_attention: blocks must be positive, max_blocks, prefix_length and window not negative");
  // the running maximum follows scores that grow with q . k
  if (!(d->scale > 0.0f) || d->scale > 3.0e38f)
    return report(Q3S_ERR_UNSUPPORTED, "q3s_chunk_attention: scale must be positive and finite");
  if (static_cast<int64_t>(d->tokens) * d->q_heads > 0x7fffffffll - 65536 ||
      static_cast<int64_t>(d->max_blocks) * d->block_size + d->prefix_length > 0x7fffffffll - 65536)
    return report(Q3S_ERR_UNSUPPORTED,
                  "q3s_chunk_attention: tokens * q_heads, and a table's tokens with prefix_length, stay below 2^31 - 2^16");
  return Q3S_OK;
}

// Whether the kernels of q3s_prefix_attention, whose tiles are 16 query rows, are the faster ones: few query rows, together or
// a row of the batch, and no window.  They against the kernel here, us, 8 key/value heads of 128, query rows a row of the
// batch: 1 row of 8000 keys, 64: 31 and 36, 128: 43 and 39, 256: 78 and 43; 1 row of 200 keys, 128: 14 and 17, 512: 24 and 21;
// 16 rows of 2000 keys, 15: 33 and 38, 31: 49 and 39; 64 rows of 1000 keys, 15: 52 and 59, 31: 82 and 60; 16 rows of 8000
// keys, 7: 71 and 77, 15: 86 and 80; 4 heads of 64, 16 rows of 2000 keys, 15: 15 and 22, 63: 29 and 23.
// The host knows the totals alone.  256 rows of 4000 keys, 2048 query rows: 8 each 664 and 827; half of them in one row, 4
// in each of the others 697 and 1013; all in one row, the others without tokens 401 and 59.  A bound on the total that
// takes the last of these to the kernel here would slow the first two; the caller can leave such rows out, or ask for this
// kernel by a window that leaves nothing out.  Rows of 17 to 20 each, all alike, are two tiles there (64 rows of 1000 keys,
// 20: 84 and 76; 256 of 4000: 1336 and 858); ragged ones of that mean are not (48 rows of up to 36: 54 and 60).
bool few_queries(const q3s_chunk_attention_desc* d) {
  const int64_t G = d->q_heads / d->kv_heads;
  return d->window == 0 && G <= Q3S_MAX_QUERY_GROUP && d->tokens * G <= std::max<int64_t>(112, static_cast<int64_t>(d->batch) * 20);
}
q3s_prefix_attention_desc few_queries_desc(const q3s_chunk_attention_desc* d) {
  q3s_prefix_attention_desc p = {};
  p.struct_size = sizeof(p);
  p.batch = d->batch;
  p.tokens = d->tokens;
  p.q_heads = d->q_heads;
  p.kv_heads = d->kv_heads;
  p.dim = d->dim;
  p.block_size = d->block_size;
  p.blocks = d->blocks;
  p.elem = d->elem;
  p.max_blocks = d->max_blocks;
  p.prefix_length = d->prefix_length;
  p.scale = d->scale;
  p.q = d->q;
  p.q_token_stride = d->q_token_stride;
  p.q_head_stride = d->q_head_stride;
  p.k_cache = d->k_cache;
  p.v_cache = d->v_cache;
  p.k_block_stride = d->k_block_stride;
  p.k_head_stride = d->k_head_stride;
  p.k_place_stride = d->k_place_stride;
  p.v_block_stride = d->v_block_stride;
  p.v_head_stride = d->v_head_stride;
  p.v_place_stride = d->v_place_stride;
  p.query_offsets = d->query_offsets;
  p.block_table = d->block_table;
  p.block_table_stride = d->block_table_stride;
  p.lengths = d->lengths;
  p.prefix_blocks = d->prefix_blocks;
  p.out = d->out;
  p.out_token_stride = d->out_token_stride;
  p.out_head_stride = d->out_head_stride;
  p.lse = d->lse;
  p.workspace = d->workspace;
  p.workspace_bytes = d->workspace_bytes;
  p.error_word = d->error_word;
  p.slot_map = d->slot_map;
  return p;
}

template <int D, bool BF16>
cudaError_t launch(const q3s::ChunkArgs& c, const Layout& l, cudaStream_t st) {
  auto kernel = q3s::attn_chunk_kernel<D, BF16>;
  constexpr int smem = q3s::ChunkTile<D>::SMEM;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = q3s::allow_smem(kernel, smem, done);
  if (e != cudaSuccess) return e;
  CUtensorMap tq, tk, tv;
  if (!q3s::query_map(c.a, D, BF16, l.per_tile, &tq) || !q3s::cache_maps(c.a, D, BF16, q3s::CH_KEYS, 1, &tk, &tv)) return cudaErrorInvalidValue;
  e = q3s::launch_maybe_pdl(kernel, dim3(static_cast<unsigned>(l.ctas)), dim3(q3s::CH_NT), smem, st, true, tq, tk, tv, c);
  if (e != cudaSuccess) return e;
  const int each = (l.slot_rows + q3s::CH_JOIN_ROWS - 1) / q3s::CH_JOIN_ROWS, join = l.ctas * each;
  const int fill = (c.a.T + q3s::CH_JOIN_NT - 1) / q3s::CH_JOIN_NT;
  return q3s::launch_maybe_pdl(q3s::attn_chunk_join_kernel<D, BF16>, dim3(static_cast<unsigned>(join + fill)), dim3(q3s::CH_JOIN_NT), 0, st,
                               true, c, join, each);
}

}  // namespace

extern "C" q3s_status q3s_chunk_attention_workspace(const q3s_chunk_attention_desc* d, int64_t* bytes) {
  const q3s_status s = check_sizes(d);
  if (s != Q3S_OK) return s;
  if (!bytes) return q3s::report(Q3S_ERR_INVALID_ARGUMENT, "q3s_chunk_attention_workspace: bytes is NULL");
  if (few_queries(d)) {
    const q3s_prefix_attention_desc p = few_queries_desc(d);
    return q3s_prefix_attention_workspace(&p, bytes);
  }
  *bytes = layout_of(d).bytes;
  return q3s::report(Q3S_OK, "");
}

extern "C" q3s_status q3s_chunk_attention(const q3s_chunk_attention_desc* d, void* stream) {
  using q3s::report;
  const q3s_status s = check_sizes(d);
  if (s != Q3S_OK) return s;
  if (d->tokens == 0) return report(Q3S_OK, "");
  if (!d->q || !d->k_cache || !d->v_cache || !d->out || !d->workspace || !d->query_offsets)
    return report(Q3S_ERR_INVALID_ARGUMENT,
                  "q3s_chunk_attention: q, k_cache, v_cache, query_offsets, out and workspace are required");
  if (d->batch > 0 && (!d->lengths || (d->max_blocks > 0 && !d->block_table)))
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_chunk_attention: lengths and block_table are required");
  if (d->prefix_length > 0 && !d->prefix_blocks)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_chunk_attention: a prefix needs prefix_blocks");
  for (const void* p : {d->q, d->k_cache, d->v_cache, static_cast<const void*>(d->out), static_cast<const void*>(d->workspace)})
    if (!q3s::aligned16(p))
      return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_chunk_attention: q, caches, out and workspace must be 16-byte aligned");
  for (int64_t x : {d->q_token_stride, d->q_head_stride, d->out_token_stride, d->out_head_stride, d->k_block_stride,
                    d->k_head_stride, d->k_place_stride, d->v_block_stride, d->v_head_stride, d->v_place_stride})
    if (x % 8)
      return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_chunk_attention: strides must be multiples of 8 elements");
  if (few_queries(d)) {
    int64_t needed = 0;
    const q3s_prefix_attention_desc p = few_queries_desc(d);
    const q3s_status sized = q3s_prefix_attention_workspace(&p, &needed);
    if (sized != Q3S_OK) return sized;
    if (d->workspace_bytes >= needed) return q3s_prefix_attention(&p, stream);
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_chunk_attention: workspace of %lld bytes, %lld needed",
                  static_cast<long long>(d->workspace_bytes), static_cast<long long>(needed));
  }
  const Layout l = layout_of(d);
  if (d->workspace_bytes < l.bytes)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_chunk_attention: workspace of %lld bytes, %lld needed",
                  static_cast<long long>(d->workspace_bytes), static_cast<long long>(l.bytes));
  q3s::ChunkArgs c = {};
  q3s::AttnArgs& a = c.a;
  a.B = d->batch;
  a.T = d->tokens;
  a.Hq = d->q_heads;
  a.H = d->kv_heads;
  a.G = d->q_heads / d->kv_heads;
  a.bs = d->block_size;
  a.bs_log2 = 4;
  while ((1 << a.bs_log2) < a.bs) ++a.bs_log2;
  a.blocks = d->blocks;
  a.max_blocks = d->max_blocks;
  a.L = d->prefix_length;
  a.scale_log2 = d->scale * 1.4426950408889634f;
  a.q = d->q;
  a.k = d->k_cache;
  a.v = d->v_cache;
  a.qt = d->q_token_stride;
  a.qh = d->q_head_stride;
  a.kb = d->k_block_stride;
  a.kh = d->k_head_stride;
  a.kp = d->k_place_stride;
  a.vb = d->v_block_stride;
  a.vh = d->v_head_stride;
  a.vp = d->v_place_stride;
  a.offsets = d->query_offsets;
  a.table = d->block_table;
  a.table_stride = d->block_table_stride;
  a.lengths = d->lengths;
  a.prefix_blocks = d->prefix_blocks;
  a.out = d->out;
  a.ot = d->out_token_stride;
  a.oh = d->out_head_stride;
  a.lse = d->lse;
  a.error_word = d->error_word;
  a.slot_map = d->slot_map;
  c.per_tile = l.per_tile;
  c.window = d->window;
  c.slot_rows = l.slot_rows;
  unsigned char* ws = static_cast<unsigned char*>(d->workspace);
  c.cuts = reinterpret_cast<q3s::ChunkCut*>(ws + l.cuts);
  c.part_ml = reinterpret_cast<float2*>(ws + l.part_ml);
  c.part_o = reinterpret_cast<float*>(ws + l.part_o);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf16 = d->elem == Q3S_ELEM_BF16;
  const cudaError_t e = d->dim == 64 ? (bf16 ? launch<64, true>(c, l, st) : launch<64, false>(c, l, st))
                                     : (bf16 ? launch<128, true>(c, l, st) : launch<128, false>(c, l, st));
  if (e != cudaSuccess) return report(Q3S_ERR_CUDA, "q3s_chunk_attention: launch failed: %s", cudaGetErrorString(e));
  return report(Q3S_OK, "");
}
