// q3s_attn.cuh -- attention over a paged cache for a batch that shares a
// prefix: the key-split kernel (every row's own tokens, and the prefix for few
// queries) and the kernel that joins the parts.
//
// With scores s_j = scale * q . k_j, any split of the keys into parts p with
//   m_p = max s_j,  l_p = sum exp(s_j - m_p),  o_p = sum exp(s_j - m_p) v_j
// joins exactly: m = max m_p, out = (sum e^(m_p - m) o_p) / (sum e^(m_p - m) l_p).
// So the prefix is computed once for all queries of the batch, and a row's own
// tokens are cut wherever that balances the GPU.  All of m, l and o are fp32;
// scores are held times log2(e) and the exponentials are ex2.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "q3s_args.cuh"
#include "q3s_decode.h"
#include "q3s_device.cuh"
#include "q3s_head.cuh"
#include "q3s_pdl.cuh"

namespace q3s {

// Keys of a unit (one pipeline stage): 4 KB of K and of V, taken 16 at a time.
template <int D>
constexpr int AT_KEYS = D == 64 ? 32 : 16;
constexpr float AT_SLACK = 8.0f;  // log2 units that a running maximum may lag behind: p up to 256
constexpr int AT_MIN_UNITS = 3;  // fewest units a warp takes before another one is used

struct AttnArgs {
  int B, T, Hq, H, G, bs, bs_log2, blocks, max_blocks;
  int L;            // prefix tokens
  int tiles0;       // item tiles of the prefix (0: it is the prefix kernel's, or empty)
  int splits;       // parts of the prefix kernel (0: not used)
  int early, lead;  // CTAs of the key-split kernel that start at once, and how many units a warp of theirs takes more
  float scale_log2;
  const void *q, *k, *v;
  int64_t qt, qh, kb, kh, kp, vb, vh, vp;
  const int32_t* offsets;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lengths;
  const int32_t* prefix_blocks;
  void* out;
  int64_t ot, oh;
  float* lse;
  int32_t* error_word;
  const int64_t* slot_map;  // or null
  // workspace
  int2* items;       // [ids] {first slot, slots} of an item's parts
  float* part_o;     // [slots][R][D]
  float2* part_ml;   // [slots][R] (m in log2 units, l)
  int64_t ids, slots;  // capacities
  float* pre_o;      // [splits][T * Hq][D]
  float2* pre_ml;    // [splits][T * Hq]
};

// Row r of the work list: r = 0 is the prefix seen by all T tokens (empty
// unless it is computed here), r = b + 1 the own tokens of batch row b.  Its
// n * G query rows are cut into tiles of R; an item is a (row, kv head, tile).
struct AttnRow {
  int t0, n, len, causal;  // first token, tokens, keys; 1: token i sees keys j <= len - n + i
  int units, tiles;
};
template <int R, int KEYS>
Q3S_DEV AttnRow attn_row(const AttnArgs& a, int r) {
  AttnRow x;
  if (r == 0) {
    x.t0 = 0;
    x.n = a.tiles0 ? a.T : 0;
    x.len = a.L;
    x.causal = 0;
  } else {
    const int o0 = a.offsets[r - 1], o1 = a.offsets[r], len = a.lengths[r - 1];
    x.t0 = min(max(o0, 0), a.T);
    x.n = min(max(o1, x.t0), a.T) - x.t0;
    x.len = static_cast<int>(min(static_cast<int64_t>(max(len, 0)), static_cast<int64_t>(a.max_blocks) * a.bs));
    x.causal = 1;
  }
  x.units = x.n > 0 ? (x.len + KEYS - 1) / KEYS : 0;
  x.tiles = x.units ? (x.n * a.G + R - 1) / R : 0;
  return x;
}
// Id of a row's first item.  Ids ascend along the work list without a count
// of the items before: row b starts at (tiles of the prefix) + t0 * G / R + b
// tiles, and the next row's start is at least its tile count further.
template <int R>
Q3S_DEV int64_t attn_first_id(const AttnArgs& a, int r, const AttnRow& x) {
  return r == 0 ? 0 : (static_cast<int64_t>(a.tiles0) + x.t0 * a.G / R + (r - 1)) * a.H;
}

template <bool BF16>
Q3S_DEV void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two fp32 values rounded to nearest even, `lo` in the low half.
template <bool BF16>
Q3S_DEV uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <bool BF16>
Q3S_DEV float2 unpack2(uint32_t p) {
  if constexpr (BF16) {
    return make_float2(__uint_as_float(p << 16), __uint_as_float(p & 0xffff0000u));
  } else {
    // both at once: single conversions go through the unit that the exponentials need
    return __half22float2(*reinterpret_cast<const __half2*>(&p));
  }
}
Q3S_DEV float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
Q3S_DEV void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
Q3S_DEV void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// An 8x8 matrix of 16-bit values (lane l: row l / 4, columns 2 (l % 4) and the next), transposed.
Q3S_DEV uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
// Part of one block of a cache, all dims: slice by slice of 64 dims (128 bytes)
// a token.  Coordinates: dim 0, token `place` of the block, slice 0, head, block.
Q3S_DEV void tma_load_block(uint32_t dst, const CUtensorMap* map, int place, int h, int block, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %2, %4, %5}], [%6];" ::
          "r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(place), "r"(h), "r"(block), "r"(smem_u32(bar))
      : "memory");
}
Q3S_DEV void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Whether the phase of that parity is complete; does not wait.
Q3S_DEV bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
Q3S_DEV void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

// a / b with b > 0, by 32-bit division where both fit (the 64-bit one costs several times as much).
Q3S_HOST_DEV long long div_nonneg(long long a, long long b) {
  if (((a | b) >> 32) == 0) return static_cast<long long>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b));
  return a / b;
}

// Where a warp is in the work list.
struct AttnPos {
  int r, h, tile, u;  // row, kv head, query tile, unit of the row's keys
  AttnRow x;
};
// The next unit (true: of another item); `row_at(r)`: row r.
template <typename Rows>
Q3S_DEV bool attn_next(const AttnArgs& a, AttnPos& p, const Rows& row_at) {
  if (++p.u < p.x.units) return false;
  p.u = 0;
  if (++p.tile < p.x.tiles) return true;
  p.tile = 0;
  if (++p.h < a.H) return true;
  p.h = 0;
  do {
    if (++p.r > a.B) return true;  // past the end: never read
    p.x = row_at(p.r);
  } while (p.x.units == 0);
  return true;
}

// Shapes of the key-split kernel: four computing warps (and one that copies)
// with rings of three units, two CTAs a SM.  At dim 64 a unit is 32 keys, because
// a copy costs the same whatever its size: with 16 (four CTAs a SM) 61 rows of 4000
// keys of 2 heads took 37.4 us against 28.8, and 40 rows of 16 x 4 queries on 1000
// keys of 8 heads 85 against 57.
template <int D, int NQ>
struct SplitTile {
  static constexpr int WARPS = 4, STAGES = 3;
  static constexpr int PER_SM = 2;
  static constexpr int KEYS = AT_KEYS<D>;
  static constexpr int NT = (WARPS + 1) * 32;
  static constexpr int HALVES = D / 64;                 // 128-byte slices of a key
  static constexpr int SLICE = KEYS * 128;              // bytes of a unit's keys in one slice
  static constexpr int BYTES = HALVES * SLICE;          // a unit's keys (or values)
  static constexpr int SMEM = 1024 + WARPS * STAGES * 2 * BYTES;
};

// A part again, key by key, with p in one piece and what a query does not see
// left out instead of taken times p = 0: there an infinity or NaN in V would
// reach the queries of the part that do not see it, and an infinity times the
// lower piece of p would be NaN for those that do.  Only for the queries in
// `which`, whose sums are not finite though their scores are; one warp, queries
// in turn, D / 32 dims a lane.
template <int D, bool BF16, int R>
Q3S_DEV void attn_part_by_key(const AttnArgs& a, const AttnRow& x, int r, int h, int tile, int first_u, int last_u,
                              int64_t slot, uint32_t which, int lane) {
  constexpr int E = D / 32, KEYS = AT_KEYS<D>;
  auto dims = [&](const void* at, int64_t offset, float (&y)[E]) {
    const uint32_t* p = reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(at) + offset + lane * E);
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const float2 f = unpack2<BF16>(p[e / 2]);
      y[e] = f.x, y[e + 1] = f.y;
    }
  };
  const int32_t* blocks = r == 0 ? a.prefix_blocks : a.table + (r - 1) * a.table_stride;
#pragma unroll 1
  for (; which; which &= which - 1) {
    const int i = __ffs(which) - 1, row = tile * R + i, token = row / a.G;
    float q[E], acc[E], m = -INFINITY, l = 0.0f;
    dims(a.q, static_cast<int64_t>(x.t0 + token) * a.qt + (static_cast<int64_t>(h) * a.G + row % a.G) * a.qh, q);
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
    const int end = min((last_u + 1) * KEYS, x.causal ? x.len - x.n + token + 1 : x.len);
#pragma unroll 1
    for (int j = first_u * KEYS; j < end; ++j) {
      const int id = blocks[j >> a.bs_log2], place = j & (a.bs - 1);
      float k[E], v[E], s = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) k[e] = v[e] = 0.0f;
      if (static_cast<unsigned>(id) < static_cast<unsigned>(a.blocks)) {
        dims(a.k, id * a.kb + h * a.kh + place * a.kp, k);
        dims(a.v, id * a.vb + h * a.vh + place * a.vp, v);
      }
#pragma unroll
      for (int e = 0; e < E; ++e) s = fmaf(q[e], k[e], s);
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) s += __shfl_xor_sync(FULL, s, d);
      s *= a.scale_log2;
      const float nm = fmaxf(m, s), base = nm == -INFINITY ? 0.0f : nm, c = ex2(m - base), p = ex2(s - base);
      m = nm;
      l = l * c + p;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = acc[e] * c + p * v[e];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) a.part_o[slot * (R * D) + i * D + lane * E + e] = acc[e];
    if (lane == 0) a.part_ml[slot * R + i] = make_float2(m, l);
  }
}

// How the unit list is cut into the warps' ranges.  The CTAs that find a SM
// free start at once, the others when the prefix kernel leaves theirs: warps of
// the first `early` CTAs take `lead` units more.
struct AttnCut {
  long long all, early, more, less;  // units, early warps, an early and a late warp's units
  Q3S_DEV long long start(long long warp) const {
    return min(warp < early ? warp * more : early * more + (warp - early) * less, all);
  }
  Q3S_DEV long long warp_of(long long u) const {
    return u < early * more ? div_nonneg(u, more) : early + div_nonneg(u - early * more, less);
  }
};
Q3S_DEV AttnCut attn_cut(const AttnArgs& a, long long all, long long ctas, long long per_cta) {
  AttnCut c;
  const long long warps = ctas * per_cta, rest = all - a.early * per_cta * a.lead, least = AT_MIN_UNITS;
  c.all = all;
  c.early = a.early * per_cta;
  if (rest > 0 || c.early == 0) {
    c.less = max(div_nonneg(max(rest, 0ll) + warps - 1, warps), least);
    c.more = c.less + a.lead;
  } else {  // the early ones can do it all
    c.less = least;
    c.more = max(div_nonneg(all + c.early - 1, c.early), least);
  }
  return c;
}

// The key-split kernel.  The keys of every item are cut into units of 4 KB; all
// units of the batch form one list, cut into contiguous ranges, one a warp, so
// that rows of any lengths load the GPU evenly with no more than one part per
// item plus one per warp.  Each CTA derives the list from the device's lengths
// (one scan of the rows), so no host plan is needed and a captured graph
// follows the lengths.
//
// The computing warps work alone, each on its own range with a ring of
// its own; one more warp copies for them (lane l for warp l; TMA,
// 128-byte swizzle), because issuing a unit's copies takes a third as long as
// computing it.  What lies
// past the end of a row's last unit is cleared in V (so that nothing that lies
// there, NaN included, reaches the products) and masked in the scores; a key that some of an
// item's queries see and others do not is masked for those, and counts for nothing; where V is not finite,
// attn_part_by_key takes the part again.  Both
// products have the keys' side as the matrix instruction's M (m16n8k16):
// S^T = K Q^T, O^T += V^T P^T, with N = 8 query rows, so one query a row and its
// group of heads waste little of it.  p is carried as the sum of two 16-bit
// values: rounding it to one would be the largest error of a query that sees
// few keys.
//
// With one query a row this is bound by reading the cache (2 * G useful
// operations a byte), as long as a warp's dependent chain of a unit stays below
// the time that its 8 KB take: 6.8 TB/s while it streams (96 rows, from 4000 to 8000
// keys), 61 rows of 6000 keys of 2 x 64 (117 MB) in 29.5 us with the start and the
// join, 96 rows of 500 behind a prefix of 1500 (130 MB) in 32.4.  With 16-row items
// the chain weighs as much, and several tiles copy the same keys: 40 rows of 1 to 9
// queries x 4 heads behind a prefix of 2049 take 44.4 us, of which the bytes are 16;
// taking the products out saved 7.  Two warps sharing the copies of 32 rows took 344
// in place of 417 us at 40 rows of 5 x 4 queries on 8000 keys, and 5 more here.
//
// The running maximum may lag by 8, as in the prefix kernel, so that a unit
// mostly needs neither the maximum over the lanes nor O rescaled (52.4 to 51.5 us
// for the 40 rows).  Query rows as the instruction's M instead, with keys as N, took
// 34 us for the 96 rows before the join; copies by lanes (cp.async) in place of TMA
// 1100 clocks for 32 keys; four 2 KB copies a unit in place of two of a
// 5-dimensional map 900 clocks to issue.  The tcgen05 form, whose M is
// 128, would be nearly empty; many queries on a long prefix are the other kernel's.
template <int D, bool BF16, int NQ>
__global__ void __launch_bounds__(SplitTile<D, NQ>::NT, SplitTile<D, NQ>::PER_SM)
    attn_split_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                      const AttnArgs a) {
  using Tile = SplitTile<D, NQ>;
  constexpr int R = 8 * NQ, AT_WARPS = Tile::WARPS, AT_NT = Tile::NT, AT_STAGES = Tile::STAGES, BARS = AT_WARPS * AT_STAGES;
  constexpr int KEYS = Tile::KEYS;
  extern __shared__ __align__(1024) unsigned char at_smem[];
  __shared__ long long s_units[AT_NT + 1];
  __shared__ AttnRow s_rows[AT_NT];  // the rows, where there are no more than threads
  __shared__ __align__(8) uint64_t s_full[BARS], s_empty[BARS];
  const int t = static_cast<int>(threadIdx.x), w = t >> 5, lane = t & 31;
  if (t == 0) {
    prefetch_map(&tm_k);
    prefetch_map(&tm_v);
    for (int i = 0; i < BARS; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], 1);
    }
    fence_mbar_init();
  }
  if (!a.splits) grid_wait();  // else the prefix kernel, launched before this one, has waited for what both read
  grid_release();

  // ---- the work list: thread t sums rows [t * per, (t + 1) * per) ------------
  const int rows = a.B + 1, per = (rows + AT_NT - 1) / AT_NT;
  long long mu = 0;
  bool bad = false;
  for (int i = 0; i < per; ++i) {
    const int r = t * per + i;
    if (r >= rows) break;
    const AttnRow x = attn_row<R, KEYS>(a, r);
    mu += static_cast<long long>(x.units) * x.tiles * a.H;
    if (r > 0) bad |= a.lengths[r - 1] != x.len || a.offsets[r - 1] != x.t0 || a.offsets[r] != x.t0 + x.n;
    if (per == 1) s_rows[t] = x;
  }
  if (bad && blockIdx.x == 0 && a.error_word) atomicOr(a.error_word, Q3S_DECERR_LENGTHS);
  s_units[t + 1] = mu;
  if (t == 0) s_units[0] = 0;
  __syncthreads();
  if (w == 0) {  // inclusive scan, AT_NT / 32 values a lane
    constexpr int V = AT_NT / 32;
    long long u[V], su = 0;
#pragma unroll
    for (int k = 0; k < V; ++k) u[k] = su += s_units[1 + lane * V + k];
    long long pu = su;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long ou = __shfl_up_sync(FULL, pu, d);
      if (lane >= d) pu += ou;
    }
    pu -= su;
#pragma unroll
    for (int k = 0; k < V; ++k) s_units[1 + lane * V + k] = pu + u[k];
  }
  __syncthreads();
  const AttnCut cuts = attn_cut(a, s_units[AT_NT], gridDim.x, AT_WARPS);
  // the range of this warp, or, in the copying warp, of warp `lane`
  const int mine = w == AT_WARPS ? lane : w;
  const long long gw = static_cast<long long>(blockIdx.x) * AT_WARPS + mine;
  const long long u0 = cuts.start(gw);
  const int total = mine < AT_WARPS ? static_cast<int>(cuts.start(gw + 1) - u0) : 0;

  auto row_at = [&](int r) { return per == 1 ? s_rows[r] : attn_row<R, KEYS>(a, r); };
  AttnPos p;
  p.r = p.h = p.tile = p.u = 0;
  if (total > 0) {
    int l = 0, r = AT_NT;  // the last thread chunk that starts at or before u0
    while (r - l > 1) {
      const int m = (l + r) >> 1;
      if (s_units[m] <= u0) l = m; else r = m;
    }
    long long at = s_units[l];
    p.r = l * per;
    for (;; ++p.r) {
      p.x = row_at(p.r);
      const long long n = static_cast<long long>(p.x.units) * p.x.tiles * a.H;
      if (u0 < at + n) break;
      at += n;
    }
    const long long d = u0 - at;
    const int in = static_cast<int>(div_nonneg(d, p.x.units));  // item within the row
    p.u = static_cast<int>(d - static_cast<long long>(in) * p.x.units);
    p.h = in / p.x.tiles;
    p.tile = in - p.h * p.x.tiles;
  }
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(at_smem) + 1023) &
                                                         ~static_cast<uintptr_t>(1023)) +
                        (mine < AT_WARPS ? mine : 0) * AT_STAGES * 2 * Tile::BYTES;
  uint64_t* full = s_full + (mine < AT_WARPS ? mine : 0) * AT_STAGES;
  uint64_t* empty = s_empty + (mine < AT_WARPS ? mine : 0) * AT_STAGES;

  if (w == AT_WARPS) {
    // ---- copies: lane l for warp l -----------------------------------------------
    auto block_of = [&](const AttnPos& q, int key) {  // the cache block of a unit's key, as the table has it
      const int j = (q.u * KEYS + key) >> a.bs_log2;
      return q.r == 0 ? a.prefix_blocks[j] : a.table[(q.r - 1) * a.table_stride + j];
    };
    // a unit of more keys than a block has is two blocks, the second where it holds some of the row
    const bool halves = KEYS > 16 && a.bs < KEYS;
    auto second = [&](const AttnPos& q) { return halves && q.u * KEYS + 16 < q.x.len; };
    int next_id = total > 0 ? block_of(p, 0) : 0, next_second = total > 0 && second(p) ? block_of(p, 16) : 0;
    int fetched = 0, idle = 0;
    bool bad_block = false;
    auto copy = [&](uint32_t dst, int id, int place, uint64_t* bar) {
      const bool inside = static_cast<unsigned>(id) < static_cast<unsigned>(a.blocks);
      bad_block |= !inside;
      if (!inside) id = a.blocks;  // past the cache: reads as zeros
      tma_load_block(dst, &tm_k, place, p.h, id, bar);
      tma_load_block(dst + Tile::BYTES, &tm_v, place, p.h, id, bar);
    };
    while (fetched < total) {
      const int s = fetched % AT_STAGES;
      if (fetched >= AT_STAGES && !mbar_test(&empty[s], ((fetched / AT_STAGES) - 1) & 1)) {
        if (++idle == (1 << 24)) break;  // the warp has given up: so does its copier
        continue;
      }
      idle = 0;
      const uint32_t dst = smem_u32(ring + s * 2 * Tile::BYTES);
      const bool two = second(p);
      mbar_expect_tx(&full[s], halves && !two ? Tile::BYTES : 2 * Tile::BYTES);
      copy(dst, next_id, (p.u * KEYS) & (a.bs - 1), &full[s]);
      if (two) copy(dst + 16 * 128, next_second, 0, &full[s]);
      if (++fetched < total) {
        attn_next(a, p, row_at);
        if (second(p)) next_second = block_of(p, 16);
        next_id = block_of(p, 0);  // not looked at before the next round: its latency is not waited for
      }
    }
    if (bad_block && a.error_word) atomicOr(a.error_word, Q3S_DECERR_BLOCK_ID);
    // no copy may be in flight when the CTA leaves: wait for each stage's last one
    for (int i = max(0, fetched - AT_STAGES); i < fetched; ++i)
      (void)mbar_wait_bounded(&full[i % AT_STAGES], (i / AT_STAGES) & 1);
    __syncwarp();
    grid_wait();  // as below
    return;
  }

  // ---- products -----------------------------------------------------------------
  const int g = lane >> 2, tq = lane & 3;
  uint32_t qf[NQ][D / 16][2];
  float o[D / 16][NQ][4], m[NQ][2], l[NQ][2];
  int lim[NQ][2], low = 0;  // last key that the lane's query rows see; the lowest of the item's
  bool fresh = true, ok = true;
  int done = 0, first_u = 0;
  for (; done < total; ++done) {
    if (fresh) {  // a new item: its queries
      fresh = false;
      first_u = p.u;
      const int M = p.x.n * a.G, r0 = p.tile * R;
      auto limit = [&](int row) { return p.x.causal ? min(p.x.len - p.x.n + row / a.G, p.x.len - 1) : p.x.len - 1; };
      low = limit(r0);
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        const int row = r0 + 8 * q + g;
        const uint16_t* src = static_cast<const uint16_t*>(a.q) + static_cast<int64_t>(p.x.t0 + row / a.G) * a.qt +
                              (static_cast<int64_t>(p.h) * a.G + row % a.G) * a.qh + 2 * tq;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          qf[q][k][0] = row < M ? *reinterpret_cast<const uint32_t*>(src + 16 * k) : 0u;
          qf[q][k][1] = row < M ? *reinterpret_cast<const uint32_t*>(src + 16 * k + 8) : 0u;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          lim[q][e] = limit(r0 + 8 * q + 2 * tq + e);
          m[q][e] = -INFINITY;
          l[q][e] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[i][q][0] = o[i][q][1] = o[i][q][2] = o[i][q][3] = 0.0f;
      }
    }
    const int st = done % AT_STAGES;
    if (lane == 0) ok = mbar_wait_bounded(&full[st], (done / AT_STAGES) & 1);
    ok = __shfl_sync(FULL, ok, 0);
    if (!ok) break;
    unsigned char* kt = ring + st * 2 * Tile::BYTES;
    const int unit0 = p.u * KEYS, valid = p.x.len - unit0;
    if (valid < KEYS) {  // clear V past the end
      for (int c = lane; c < (KEYS - valid) * 8; c += 32)
#pragma unroll
        for (int x = 0; x < Tile::HALVES; ++x)
          *reinterpret_cast<uint4*>(kt + Tile::BYTES + x * Tile::SLICE + valid * 128 + c * 16) = make_uint4(0, 0, 0, 0);
      fence_proxy_async_smem();  // the next copy into this stage comes after
      __syncwarp();
    }
#pragma unroll
    for (int part = 0; part < KEYS / 16; ++part) {
      if (part && valid <= 16 * part) break;
      const int j0 = unit0 + 16 * part;
      const uint32_t ka = smem_u32(kt) + part * 16 * 128, va = ka + Tile::BYTES;

      float s[2][NQ][4];  // two chains of sums, over every other 16 dims
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int q = 0; q < NQ; ++q) s[i][q][0] = s[i][q][1] = s[i][q][2] = s[i][q][3] = 0.0f;
      {
        // the four 8x8 matrices: keys (lane & 7) + 8 ((lane >> 3) & 1), 16-byte chunk + (lane >> 4)
        const int key = (lane & 7) + (((lane >> 3) & 1) << 3), cc = lane >> 4, x7 = key & 7;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          uint32_t f[4];
          ldsm4(f, ka + static_cast<uint32_t>((k / 4) * Tile::SLICE + key * 128 + ((((2 * k) & 7) + cc) ^ x7) * 16));
#pragma unroll
          for (int q = 0; q < NQ; ++q) mma16816<BF16>(s[k & 1][q], f, qf[q][k][0], qf[q][k][1]);
        }
      }
      const bool cut = j0 + 15 > low;
      // a lane looks at its own scores only; what rises above the maximum by more than the slack moves it
      float top[NQ][2];
      bool rise = false;
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[0][q][e] = (s[0][q][e] + s[1][q][e]) * a.scale_log2;
          if (cut && j0 + g + 8 * (e >> 1) > lim[q][e & 1]) s[0][q][e] = -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[q][e] = fmaxf(s[0][q][e], s[0][q][2 + e]);
          rise |= top[q][e] > m[q][e] + AT_SLACK;
        }
      }
      if (__any_sync(FULL, rise)) {
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          float c[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top[q][e] = fmaxf(top[q][e], __shfl_xor_sync(FULL, top[q][e], d));
            const float nm = fmaxf(m[q][e], top[q][e]);
            c[e] = ex2(m[q][e] - (nm == -INFINITY ? 0.0f : nm));  // 0 for the item's first unit (m = -inf)
            m[q][e] = nm;
            l[q][e] *= c[e];
          }
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            o[i][q][0] *= c[0];
            o[i][q][1] *= c[1];
            o[i][q][2] *= c[0];
            o[i][q][3] *= c[1];
          }
        }
      }
      float base[NQ][2];
#pragma unroll
      for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int e = 0; e < 2; ++e) base[q][e] = m[q][e] == -INFINITY ? 0.0f : m[q][e];
      uint32_t ph[NQ][2], pl[NQ][2];  // p^T, upper and lower part: the B operand
#pragma unroll
      for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p0 = ex2(s[0][q][2 * e] - base[q][0]), p1 = ex2(s[0][q][2 * e + 1] - base[q][1]);
          l[q][0] += p0;
          l[q][1] += p1;
          const uint32_t hi = pack2<BF16>(p0, p1);
          const float2 back = unpack2<BF16>(hi);
          ph[q][e] = transpose8(hi);
          pl[q][e] = transpose8(pack2<BF16>(p0 - back.x, p1 - back.y));
        }
      {
        // V^T: keys (lane & 7) + 8 (lane >> 4), 16-byte chunk + ((lane >> 3) & 1)
        const int key = (lane & 7) + ((lane >> 4) << 3), cc = (lane >> 3) & 1, x7 = key & 7;
        constexpr int GROUP = 4 / NQ;  // dims whose products stand between the two that add to one sum
#pragma unroll
        for (int d0 = 0; d0 < D / 16; d0 += GROUP) {
          uint32_t f[GROUP][4];
#pragma unroll
          for (int d = 0; d < GROUP; ++d)
            ldsm4t(f[d], va + static_cast<uint32_t>(((d0 + d) / 4) * Tile::SLICE + key * 128 + ((((2 * (d0 + d)) & 7) + cc) ^ x7) * 16));
#pragma unroll
          for (int d = 0; d < GROUP; ++d)
#pragma unroll
            for (int q = 0; q < NQ; ++q) mma16816<BF16>(o[d0 + d][q], f[d], ph[q][0], ph[q][1]);
#pragma unroll
          for (int d = 0; d < GROUP; ++d)
#pragma unroll
            for (int q = 0; q < NQ; ++q) mma16816<BF16>(o[d0 + d][q], f[d], pl[q][0], pl[q][1]);
        }
      }
    }
    __syncwarp();  // every lane has read the stage
    if (lane == 0) mbar_arrive(&empty[st]);

    const int wr = p.r, wh = p.h, wt = p.tile, wu = p.u;
    const AttnRow wx = p.x;
    const bool last = done + 1 == total;
    if (attn_next(a, p, row_at) || last) {  // the warp's part of this item is complete
      fresh = true;
      const int64_t id = attn_first_id<R>(a, wr, wx) + static_cast<int64_t>(wh) * wx.tiles + wt;
      const int64_t slot = gw + id;
      const int M = wx.n * a.G - wt * R;
      if (slot < a.slots && id < a.ids) {
        if (first_u == 0 && lane == 0) {
          int parts = 1;
          if (wu + 1 < wx.units)  // it goes on in other warps' ranges
            parts = static_cast<int>(cuts.warp_of(u0 + done + (wx.units - 1 - wu)) - gw) + 1;
          a.items[id] = make_int2(static_cast<int>(slot), parts);
        }
        float* po = a.part_o + slot * (R * D);
        uint32_t odd = 0;  // query rows whose sums are not finite, though the sum of their p is
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = l[q][e];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) x += __shfl_xor_sync(FULL, x, d);
            const int row = 8 * q + 2 * tq + e;
            float size = x * 0.0f;  // 0, and NaN once something is not finite
            const bool known = size == 0.0f;
            if (row < M) {
#pragma unroll
              for (int i = 0; i < D / 16; ++i) {
                po[row * D + 16 * i + g] = o[i][q][e];
                po[row * D + 16 * i + g + 8] = o[i][q][2 + e];
                size = fmaf(o[i][q][e], 0.0f, fmaf(o[i][q][2 + e], 0.0f, size));
              }
              if (g == 0) a.part_ml[slot * R + row] = make_float2(m[q][e], x);
            }
            const uint32_t lanes = __ballot_sync(FULL, row < M && known && size != 0.0f);
#pragma unroll
            for (int d = 0; d < 4; ++d)  // lanes d, d + 4, .. hold row 8 q + 2 d + e
              if (lanes & (0x11111111u << d)) odd |= 1u << (8 * q + 2 * d + e);
          }
        if (odd) {
          __syncwarp();  // its writes come after those above
          attn_part_by_key<D, BF16, R>(a, wx, wr, wh, wt, first_u, wu, slot, odd, lane);
        }
      }
    }
  }
  if (!ok && lane == 0 && a.error_word) atomicOr(a.error_word, Q3S_DECERR_WAIT);  // a copy did not arrive
  // this grid starts beside the prefix kernel's: it does not end before that
  // one, so that the join, which waits for this grid, has both
  grid_wait();
}

// Joins the parts of each query row (m, l, o as above) and writes out and lse.
// One warp a row of [T * q_heads]; a lane holds D / 32 of its values.  A token's batch row is found in
// query_offsets by bisection, before the grid waits for the parts; tokens past
// the last row, and those of a refused row (slot_map), see nothing.  Bound by latency, of the record of the row's own
// parts and of the sums, and by fetching its own instructions: kept short (with the weights of
// up to 32 parts computed before the sums it took 8.8 us, and 256 rows of 32 heads
// 99 us in all against 93).
//
// TEAM: the four warps of a CTA share a row, each every fourth part, and meet in
// shared memory.
template <int D, bool BF16, int R, bool TEAM>
__global__ void __launch_bounds__(128) attn_join_kernel(const AttnArgs a) {
  constexpr int E = D / 32, AHEAD = 4, STRIDE = TEAM ? 4 : 1;
  const int lane = static_cast<int>(threadIdx.x) & 31, w = static_cast<int>(threadIdx.x) >> 5;
  const int64_t out_row = TEAM ? static_cast<int64_t>(blockIdx.x) : static_cast<int64_t>(blockIdx.x) * 4 + w;
  const int token = static_cast<int>(out_row / a.Hq), head = static_cast<int>(out_row - static_cast<int64_t>(token) * a.Hq);
  const int h = head / a.G, gq = head - h * a.G;
  AttnRow x;
  x.units = 0;
  bool live = false;
  int b = 0;
  if (token < a.T && a.B > 0) {
    int r = a.B;  // offsets[b] <= token < offsets[r], once it is known that there is such a row
    while (r - b > 1) {
      const int m = (b + r) >> 1;
      if (a.offsets[m] <= token) b = m; else r = m;
    }
    x = attn_row<R, AT_KEYS<D>>(a, b + 1);
    live = token >= x.t0 && token < x.t0 + x.n && (!a.slot_map || a.slot_map[token] >= 0);
    if (!live) x.units = 0;
  }
  grid_wait();
  grid_release();
  if (token >= a.T) return;
  {
    const int row = live ? (token - x.t0) * a.G + gq : 0;  // of the batch row's n * G
    int2 own = make_int2(0, 0);
    if (x.units) {
      const int64_t id = attn_first_id<R>(a, b + 1, x) + static_cast<int64_t>(h) * x.tiles + row / R;
      if (id < a.ids) own = a.items[id];
    }
    float acc[E], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
    // n parts: query row `at + i * step` of `o` and `ml`, in order, AHEAD of them requested at a time
    auto join = [&](const float* o, const float2* ml, int64_t at, int64_t step, int n) {
      if constexpr (TEAM) {  // this warp's
        at += w * step;
        step *= STRIDE;
        n = (n - w + STRIDE - 1) / STRIDE;
      }
      const float* src = o + at * D + lane * E;
      const float2* sml = ml + at;
      for (int i = 0; i < n; i += AHEAD) {
        float y[AHEAD][E];
        float2 p[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          p[k] = make_float2(-INFINITY, 0.0f);
          if (i + k < n) {
            p[k] = *sml;
            if constexpr (E == 4) {
              const float4 f = *reinterpret_cast<const float4*>(src);
              y[k][0] = f.x, y[k][1] = f.y, y[k][2] = f.z, y[k][3] = f.w;
            } else {
              const float2 f = *reinterpret_cast<const float2*>(src);
              y[k][0] = f.x, y[k][1] = f.y;
            }
          }
          src += step * D;
          sml += step;
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          if (i + k >= n) break;
          const float nm = fmaxf(m, p[k].x), base = nm == -INFINITY ? 0.0f : nm;
          const float c = ex2(m - base), wt = ex2(p[k].x - base);
          m = nm;
          l = l * c + wt * p[k].y;
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] = acc[e] * c + wt * y[k][e];
        }
      }
    };
    auto parts = [&](int2 it) { return it.x >= 0 && it.y > 0 && static_cast<int64_t>(it.x) + it.y <= a.slots ? it.y : 0; };
    if (live && a.tiles0) {
      const int r = token * a.G + gq;
      const int2 it = a.items[static_cast<int64_t>(h) * a.tiles0 + r / R];
      join(a.part_o, a.part_ml, static_cast<int64_t>(it.x) * R + r % R, R, parts(it));
    } else if (live && a.splits) {
      join(a.pre_o, a.pre_ml, out_row, static_cast<int64_t>(a.T) * a.Hq, a.splits);
    }
    join(a.part_o, a.part_ml, static_cast<int64_t>(own.x) * R + row % R, R, parts(own));
    if constexpr (TEAM) {
      __shared__ float s_acc[3][32][E + 1], s_ml[3][2];
      if (w) {
#pragma unroll
        for (int e = 0; e < E; ++e) s_acc[w - 1][lane][e] = acc[e];
        if (lane == 0) s_ml[w - 1][0] = m, s_ml[w - 1][1] = l;
      }
      __syncthreads();
      if (w) return;
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        const float nm = fmaxf(m, s_ml[k][0]), base = nm == -INFINITY ? 0.0f : nm;
        const float c = ex2(m - base), wt = ex2(s_ml[k][0] - base);
        m = nm;
        l = l * c + wt * s_ml[k][1];
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = acc[e] * c + wt * s_acc[k][lane][e];
      }
    }
    const float inv = l > 0.0f ? 1.0f / l : l == l ? 0.0f : l;  // a NaN stays one
    uint16_t* dst = static_cast<uint16_t*>(a.out) + token * a.ot + head * a.oh + lane * E;
    if constexpr (E == 4)
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<BF16>(acc[0] * inv, acc[1] * inv), pack2<BF16>(acc[2] * inv, acc[3] * inv));
    else
      *reinterpret_cast<uint32_t*>(dst) = pack2<BF16>(acc[0] * inv, acc[1] * inv);
    if (a.lse && lane == 0)
      a.lse[out_row] =
          l > 0.0f ? (m + log2f(l)) * 0.69314718055994531f : l == l ? -INFINITY : l;
  }
}

}  // namespace q3s
