// q3s_attn.cu -- host side of q3s_prefix_attention.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstring>

#include "q3s_attn.cuh"
#include "q3s_tma.cuh"

namespace {

constexpr int kSplitThreads = q3s::AT_WARPS * 32;

int split_smem(int dim) { return q3s::AT_WARPS * q3s::AT_STAGES * 2 * q3s::AT_KEYS * dim * 2; }
// CTAs of the key-split kernel: as many as are resident
int split_ctas(int dim) { return q3s::sm_count() * ((227 * 1024) / (split_smem(dim) + 4096)); }

struct Layout {
  int64_t plan, part_o, part_ml, pre_o, pre_ml, bytes;  // byte offsets
  int64_t slots;
  int ctas, splits;
  bool prefix_here;
};

Layout layout_of(const q3s_prefix_attention_desc* d) {
  Layout l;
  const int64_t G = d->q_heads / d->kv_heads, queries = static_cast<int64_t>(d->tokens) * G;
  l.prefix_here = true;
  l.splits = 0;
  l.ctas = split_ctas(d->dim);
  const int64_t items = (queries + q3s::AT_ROWS - 1) / q3s::AT_ROWS * (l.prefix_here ? 1 : 0) + queries / q3s::AT_ROWS +
                        std::min<int64_t>(d->batch, d->tokens);
  l.slots = items * d->kv_heads + static_cast<int64_t>(l.ctas) * q3s::AT_WARPS;
  auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
  int64_t at = 0;
  l.plan = at;
  at += up(12 * (static_cast<int64_t>(d->batch) + 2) + 8);
  l.part_ml = at;
  at += up(l.slots * q3s::AT_ROWS * 8);
  l.part_o = at;
  at += up(l.slots * q3s::AT_ROWS * d->dim * 4);
  l.pre_ml = at;
  at += up(static_cast<int64_t>(l.splits) * d->tokens * d->q_heads * 8);
  l.pre_o = at;
  at += up(static_cast<int64_t>(l.splits) * d->tokens * d->q_heads * d->dim * 4);
  l.bytes = at;
  return l;
}

q3s_status check_sizes(const q3s_prefix_attention_desc* d) {
  using q3s::report;
  if (!d) return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_prefix_attention: desc is NULL");
  if (d->struct_size != sizeof(q3s_prefix_attention_desc))
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_prefix_attention: struct_size %u != %u (ABI mismatch)", d->struct_size,
                  static_cast<unsigned>(sizeof(q3s_prefix_attention_desc)));
  if (d->batch < 0 || d->batch > Q3S_MAX_CACHE_ROWS || d->tokens < 0)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_prefix_attention: batch %d is not in [0, %d] or tokens %d is negative",
                  d->batch, Q3S_MAX_CACHE_ROWS, d->tokens);
  if (d->kv_heads < 1 || d->q_heads < 1 || d->q_heads % d->kv_heads || d->q_heads / d->kv_heads > Q3S_MAX_QUERY_GROUP)
    return report(Q3S_ERR_INVALID_ARGUMENT,
                  "q3s_prefix_attention: %d query heads are not 1 to %d for each of %d key/value heads", d->q_heads,
                  Q3S_MAX_QUERY_GROUP, d->kv_heads);
  if (d->kv_heads > 65535)
    return report(Q3S_ERR_UNSUPPORTED, "q3s_prefix_attention: %d key/value heads are too many", d->kv_heads);
  if (d->dim != 64 && d->dim != 128)
    return report(Q3S_ERR_UNSUPPORTED, "q3s_prefix_attention: dim %d is not 64 or 128", d->dim);
  if (d->block_size != 16 && d->block_size != 32 && d->block_size != 64 && d->block_size != 128)
    return report(Q3S_ERR_UNSUPPORTED, "q3s_prefix_attention: block_size %d is not 16, 32, 64 or 128", d->block_size);
  if (d->elem != Q3S_ELEM_BF16 && d->elem != Q3S_ELEM_F16)
    return report(Q3S_ERR_UNSUPPORTED, "q3s_prefix_attention: elem %d is not bf16 or f16", d->elem);
  if (d->blocks < 1 || d->max_blocks < 0 || d->prefix_length < 0)
    return report(Q3S_ERR_INVALID_ARGUMENT,
                  "q3s_prefix_attention: blocks must be positive, max_blocks and prefix_length not negative");
  if (static_cast<int64_t>(d->tokens) * d->q_heads > 0x7fffffffll - 65536 ||
      static_cast<int64_t>(d->max_blocks) * d->block_size > 0x7fffffffll - 65536 || d->prefix_length > 0x7fffffff - 65536)
    return report(Q3S_ERR_UNSUPPORTED, "q3s_prefix_attention: tokens * q_heads, a table's tokens and prefix_length stay below 2^31 - 2^16");
  return Q3S_OK;
}

template <int D, bool BF16>
cudaError_t launch(const q3s::AttnArgs& a, const Layout& l, cudaStream_t st) {
  auto split = q3s::attn_split_kernel<D, BF16>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = q3s::allow_smem(split, split_smem(D), done);
  if (e != cudaSuccess) return e;
  split<<<l.ctas, kSplitThreads, split_smem(D), st>>>(a);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  // a warp joins one query row: rows of a (row, head) spread over gridDim.z CTAs of 4 warps
  const int64_t per = (static_cast<int64_t>(a.T) * a.G + a.B - 1) / std::max(a.B, 1);
  const int z = static_cast<int>(std::min<int64_t>(64, std::max<int64_t>(1, (per + 3) / 4)));
  return q3s::launch_maybe_pdl(q3s::attn_join_kernel<D, BF16>, dim3(a.B + 1, a.H, z), dim3(128), 0, st, true, a);
}

}  // namespace

extern "C" q3s_status q3s_prefix_attention_workspace(const q3s_prefix_attention_desc* d, int64_t* bytes) {
  const q3s_status s = check_sizes(d);
  if (s != Q3S_OK) return s;
  if (!bytes) return q3s::report(Q3S_ERR_INVALID_ARGUMENT, "q3s_prefix_attention_workspace: bytes is NULL");
  *bytes = layout_of(d).bytes;
  return q3s::report(Q3S_OK, "");
}

extern "C" q3s_status q3s_prefix_attention(const q3s_prefix_attention_desc* d, void* stream) {
  using q3s::report;
  const q3s_status s = check_sizes(d);
  if (s != Q3S_OK) return s;
  if (d->tokens == 0) return report(Q3S_OK, "");
  if (!d->q || !d->k_cache || !d->v_cache || !d->out || !d->workspace || !d->query_offsets)
    return report(Q3S_ERR_INVALID_ARGUMENT,
                  "q3s_prefix_attention: q, k_cache, v_cache, query_offsets, out and workspace are required");
  if (d->batch > 0 && (!d->lengths || (d->max_blocks > 0 && !d->block_table)))
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_prefix_attention: lengths and block_table are required");
  if (d->prefix_length > 0 && !d->prefix_blocks)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_prefix_attention: a prefix needs prefix_blocks");
  for (const void* p : {d->q, d->k_cache, d->v_cache, static_cast<const void*>(d->out), static_cast<const void*>(d->workspace)})
    if (!q3s::aligned16(p))
      return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_prefix_attention: q, caches, out and workspace must be 16-byte aligned");
  for (int64_t x : {d->q_token_stride, d->q_head_stride, d->out_token_stride, d->out_head_stride, d->k_block_stride,
                    d->k_head_stride, d->k_place_stride, d->v_block_stride, d->v_head_stride, d->v_place_stride})
    if (x % 8)
      return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_prefix_attention: strides must be multiples of 8 elements");
  const Layout l = layout_of(d);
  if (d->workspace_bytes < l.bytes)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_prefix_attention: workspace of %lld bytes, %lld needed",
                  static_cast<long long>(d->workspace_bytes), static_cast<long long>(l.bytes));
  q3s::AttnArgs a;
  a.B = d->batch;
  a.T = d->tokens;
  a.Hq = d->q_heads;
  a.H = d->kv_heads;
  a.G = d->q_heads / d->kv_heads;
  a.bs = d->block_size;
  a.blocks = d->blocks;
  a.max_blocks = d->max_blocks;
  a.L = d->prefix_length;
  a.prefix_here = l.prefix_here;
  a.splits = l.splits;
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
  unsigned char* ws = static_cast<unsigned char*>(d->workspace);
  a.plan = reinterpret_cast<int32_t*>(ws + l.plan);
  a.part_o = reinterpret_cast<float*>(ws + l.part_o);
  a.part_ml = reinterpret_cast<float2*>(ws + l.part_ml);
  a.slots = l.slots;
  a.pre_o = reinterpret_cast<float*>(ws + l.pre_o);
  a.pre_ml = reinterpret_cast<float2*>(ws + l.pre_ml);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf16 = d->elem == Q3S_ELEM_BF16;
  const cudaError_t e = d->dim == 64 ? (bf16 ? launch<64, true>(a, l, st) : launch<64, false>(a, l, st))
                                     : (bf16 ? launch<128, true>(a, l, st) : launch<128, false>(a, l, st));
  if (e != cudaSuccess) return report(Q3S_ERR_CUDA, "q3s_prefix_attention: launch failed: %s", cudaGetErrorString(e));
  return report(Q3S_OK, "");
}
