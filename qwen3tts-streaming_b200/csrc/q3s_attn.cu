// q3s_attn.cu -- host side of q3s_prefix_attention.
#include <cuda.h>
#include <cuda_runtime.h>
#include <stddef.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>

#include "q3s_attn.cuh"
#include "q3s_attn_maps.cuh"
#include "q3s_attn_prefix.cuh"
#include "q3s_tma.cuh"

namespace {

// Computing warps of the key-split kernel's grid.
int split_warps() { return q3s::sm_count() * q3s::SplitTile<128, 1>::PER_SM * q3s::SplitTile<128, 1>::WARPS; }

struct Layout {
  int64_t items, part_o, part_ml, pre_o, pre_ml, bytes;  // byte offsets
  int64_t ids, slots;
  int nq;      // 8-row query tiles of an item of the key-split kernel: 1 or 2
  int tiles0;  // tiles of the prefix there (0: none)
  int early, lead;
  int per_tile, pairs, steps, per_split, splits;  // the prefix kernel's (splits 0: not used)
};

// Parts that the prefix kernel cuts the keys into.  A part costs its steps of
// 128 keys plus about three for its start and end; the CTAs of all parts run
// in waves of one a SM; each part writes and the join reads fp32 sums of all
// queries; and the SMs that the CTAs hold are time that the key-split kernel
// beside them does not have, which weighs more where that one has 16-row items
// (without the term 40 ragged rows took 6 parts and 51.6 us, with it 3 and 43.9;
// 96 rows 6 and 32.6, 4 and 31.8; at the full weight 32 rows with short caches
// behind 2048 keys took 18.1 us in place of 15.2).  The number with the lowest
// estimate is taken.
void plan_prefix(const q3s_prefix_attention_desc* d, Layout* l) {
  const int G = d->q_heads / d->kv_heads;
  l->per_tile = q3s::PX_M / G;
  l->pairs = (d->tokens + 2 * l->per_tile - 1) / (2 * l->per_tile);
  l->steps = (d->prefix_length + q3s::PX_KEYS - 1) / q3s::PX_KEYS;
  const int64_t items = static_cast<int64_t>(l->pairs) * d->kv_heads, sms = q3s::sm_count();
  const double step_us = 1.6, part_us = 0.5 + static_cast<double>(d->tokens) * d->q_heads * d->dim * 8 / 6e6;
  double best = 0;
  for (int s = 1; s <= l->steps && s <= 64; ++s) {
    const int per = (l->steps + s - 1) / s, parts = (l->steps + per - 1) / per;
    if (parts != s) continue;
    const double part = (per + 3) * step_us, held = static_cast<double>(items * s) / sms;
    const double cost = (std::ceil(held) + (l->nq == 1 ? 0.4 : 1.0) * held) * part + s * part_us;
    if (l->splits == 0 || cost < best) {
      best = cost;
      l->splits = s;
      l->per_split = per;
    }
  }
}

Layout layout_of(const q3s_prefix_attention_desc* d) {
  Layout l;
  const int64_t G = d->q_heads / d->kv_heads, queries = static_cast<int64_t>(d->tokens) * G;
  // An item of the key-split kernel holds the query rows of an average row of
  // the batch (an item reads its keys once), in tiles of 8 or 16.  8 against 16,
  // 60 rows of 2000 keys: 8 query rows 85 against 93 us, 10 query rows 160
  // against 95; 16 rows of 1000 keys: 13.4 against 17.7 and 19.0 against 18.1.
  const int64_t mean = (queries + std::max(d->batch, 1) - 1) / std::max(d->batch, 1);
  l.nq = mean <= 8 ? 1 : 2;
  // With few queries or keys the key-split kernel takes the prefix as one more
  // row: that costs it about queries * keys, the prefix kernel about the square
  // root of the keys (more of them are cut into more parts).  So the rule is on
  // queries^2 * keys.  Key-split against prefix kernel, 8 heads of 128 and 100
  // own tokens: 32 queries x 2048 keys (2.1e6) 14.0 against 15.2 us, 32 x 8192
  // (8.4e6) 22.6 against 20.9, 48 x 2048 (4.7e6) 15.0 against 15.6, 64 x 2048
  // (8.4e6) 16.8 against 15.6, 128 x 128 (2.1e6) 11.4 to 12.2 against 12.5 to 13.4,
  // 96 x 512 (4.7e6) 14.4 against 13.0, 256 x 8192 106 to 110 against 28 to 32.  A scale that is not positive turns the order of the scores
  // around, which the prefix kernel's running maximum does not follow.
  l.splits = 0;
  if (queries * queries >= 4000000 / std::max(d->prefix_length, 1) && d->prefix_length >= 64 && d->scale > 0.0f) plan_prefix(d, &l);
  const int64_t warps = split_warps();
  // A CTA of the prefix kernel has a SM for itself: this kernel's CTAs that
  // would be there start when it ends, that many units later (a unit takes 1.3
  // us with 8-row items, 2 us with 16-row ones, and a CTA 3 us to get going).  With
  // 4, 8, 12 and 16 for the constant of 8-row items 96 rows take 35.0, 33.1, 32.8
  // and 32.9 us, 256 rows behind 16000 keys 90.0, 90.2, 88.3 and 90.1; with 4, 8 and 12
  // for that of 16-row ones 40 ragged rows 45.3, 43.9 and 46.8.
  const int64_t busy = l.splits ? std::min<int64_t>(static_cast<int64_t>(l.pairs) * d->kv_heads * l.splits, q3s::sm_count()) : 0;
  const int64_t ctas = warps / q3s::SplitTile<64, 1>::WARPS;
  l.early = static_cast<int>(ctas - busy * (ctas / q3s::sm_count()));
  l.lead = l.splits ? (l.nq == 1 ? 12 + l.per_split * 17 / 10 : 8 + l.per_split) : 0;
  const int64_t R = 8 * l.nq;
  l.tiles0 = l.splits || d->prefix_length == 0 ? 0 : static_cast<int>((queries + R - 1) / R);
  l.ids = (l.tiles0 + queries / R + d->batch + 1) * d->kv_heads;
  l.slots = l.ids + warps;
  auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
  int64_t at = 0;
  l.items = at;
  at += up(l.ids * 8);
  l.part_ml = at;
  at += up(l.slots * R * 8);
  l.part_o = at;
  at += up(l.slots * R * d->dim * 4);
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
  if (d->struct_size != sizeof(q3s_prefix_attention_desc) && d->struct_size != offsetof(q3s_prefix_attention_desc, slot_map))
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

template <int D, bool BF16, int NQ>
cudaError_t launch_split(const q3s::AttnArgs& a, cudaStream_t st) {
  using Tile = q3s::SplitTile<D, NQ>;
  auto split = q3s::attn_split_kernel<D, BF16, NQ>;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = q3s::allow_smem(split, Tile::SMEM, done);
  if (e != cudaSuccess) return e;
  CUtensorMap tk, tv;
  if (!q3s::cache_maps(a, D, BF16, Tile::KEYS, D / 64, &tk, &tv)) return cudaErrorInvalidValue;
  return q3s::launch_maybe_pdl(split, dim3(q3s::sm_count() * Tile::PER_SM), dim3(Tile::NT), Tile::SMEM, st, true, tk, tv, a);
}

// A warp a row, or four where an item is cut into many parts (few items over
// all the warps, or many parts of the prefix).  One against four, 8 heads, rows
// of 2000 keys: 1 row 14.0 against 10.1 us, 24 rows 40.5 against 38.6, 48 rows
// 71.1 against 72.6; 64 rows, 2 heads, a prefix of 30000 in 32 parts: 34.2 against 32.1.
template <int D, bool BF16, int R>
cudaError_t launch_join(const q3s::AttnArgs& a, const Layout& l, cudaStream_t st) {
  const int64_t rows = static_cast<int64_t>(a.T) * a.Hq;
  const int64_t items = static_cast<int64_t>(std::max(std::min(a.B, a.T), 1)) * a.H;
  return l.splits > 12 || split_warps() / items >= 4
             ? q3s::launch_maybe_pdl(q3s::attn_join_kernel<D, BF16, R, true>, dim3(static_cast<unsigned>(rows)), dim3(128), 0, st, true, a)
             : q3s::launch_maybe_pdl(q3s::attn_join_kernel<D, BF16, R, false>, dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(128), 0,
                                     st, true, a);
}

template <int D, bool BF16>
cudaError_t launch_prefix(const q3s::AttnArgs& a, const Layout& l, cudaStream_t st) {
  auto prefix = q3s::attn_prefix_kernel<D, BF16>;
  constexpr int smem = q3s::PrefixTile<D>::SMEM;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = q3s::allow_smem(prefix, smem, done);
  if (e != cudaSuccess) return e;
  CUtensorMap tq, tk, tv;
  if (!q3s::query_map(a, D, BF16, l.per_tile, &tq) || !q3s::cache_maps(a, D, BF16, q3s::PX_KEYS, 1, &tk, &tv)) return cudaErrorInvalidValue;
  q3s::PrefixArgs p;
  p.a = a;
  p.per_tile = l.per_tile;
  p.steps = l.steps;
  p.per_split = l.per_split;
  return q3s::launch_maybe_pdl(prefix, dim3(l.pairs, a.H, l.splits), dim3(q3s::PX_NT), smem, st, true, tq, tk, tv, p);
}

template <int D, bool BF16>
cudaError_t launch(const q3s::AttnArgs& a, const Layout& l, cudaStream_t st) {
  cudaError_t e = l.splits ? launch_prefix<D, BF16>(a, l, st) : cudaSuccess;
  if (e != cudaSuccess) return e;
  // beside the prefix kernel where there is one: neither reads what the other writes
  e = l.nq == 1 ? launch_split<D, BF16, 1>(a, st) : launch_split<D, BF16, 2>(a, st);
  if (e != cudaSuccess) return e;
  return l.nq == 1 ? launch_join<D, BF16, 8>(a, l, st) : launch_join<D, BF16, 16>(a, l, st);
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
  a.bs_log2 = 4;
  while ((1 << a.bs_log2) < a.bs) ++a.bs_log2;
  a.blocks = d->blocks;
  a.max_blocks = d->max_blocks;
  a.L = d->prefix_length;
  a.tiles0 = l.tiles0;
  a.splits = l.splits;
  a.early = l.early;
  a.lead = l.lead;
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
  a.slot_map = d->struct_size == sizeof(q3s_prefix_attention_desc) ? d->slot_map : nullptr;
  unsigned char* ws = static_cast<unsigned char*>(d->workspace);
  a.items = reinterpret_cast<int2*>(ws + l.items);
  a.part_o = reinterpret_cast<float*>(ws + l.part_o);
  a.part_ml = reinterpret_cast<float2*>(ws + l.part_ml);
  a.ids = l.ids;
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
