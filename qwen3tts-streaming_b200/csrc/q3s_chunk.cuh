// q3s_chunk.cuh -- attention of every row's chunk of new tokens over its pages
// (q3s_chunk_attention): the tensor-core kernel and the kernel that joins its parts.
//
// An item is a key/value head and up to 256 query rows (two tiles of 128) of one
// row of the batch: query rows are (token, head of the group) pairs, so a group's
// heads share the keys that are read.  Its keys are taken in steps of 128: first the
// steps of the prefix, then those of the row's own tokens, from the first that a query of the item sees to the last.
//
// All steps of all items form one list, which the CTAs cut into equal ranges (by
// an estimate of their time), one CTA a SM, so that rows of any lengths load the GPU evenly
// with at most two cut items a CTA.  Each CTA derives its range from the device's lengths, so no host
// plan is needed and a captured graph follows the lengths.  A whole item is written as
// it ends; the parts (m, l, o) of a cut one are joined by the second kernel (q3s_attn.cuh has the mathematics).
#pragma once

#include <cuda.h>

#include "q3s_attn.cuh"
#include "q3s_attn_prefix.cuh"
#include "q3s_head.cuh"

namespace q3s {

constexpr int CH_M = PX_M, CH_KEYS = PX_KEYS;
constexpr int CH_NT = 320;      // two softmax warpgroups (a tile each), the copy warp, the matrix warp
constexpr int CH_SEGS = 64;     // segments of a CTA's range that are listed at a time
constexpr int CH_START = 6;     // cost of an item's start and end, where a step of two tiles costs 3 and one of one tile 2
constexpr int CH_MAX_STEP = 3;  // the largest cost of a step
constexpr int CH_JOIN_NT = 256, CH_JOIN_ROWS = 32;  // threads and query rows of a CTA of the joining kernel

// A CTA's piece of an item.
struct ChunkSeg {
  int b, h;           // row of the batch, key/value head
  int token, tokens;  // first query token (of the packed batch), tokens
  int i_key;          // own tokens that the first query sees (its place in the row, and one)
  int len;            // own tokens of the row
  int step0, steps;   // steps of the item's list: [step0, step0 + steps)
  int slot;           // its part's place in the workspace; -1: the whole item
};

// What the joining kernel needs of an item that was cut, one for each CTA that holds the first piece of one.
struct ChunkCut {
  int parts;  // 0: no such item
  int slot;   // of the first part; the following ones are the first pieces of CTAs cta + 1, ...
  int cta;
  int h, token, tokens;
};

// First token, tokens and own tokens of a row of the batch.
struct ChunkRow {
  int t0, n, len;
};

template <int D>
struct ChunkTile {
  static constexpr int HALVES = D / 64;
  static constexpr int STAGES = D == 64 ? 4 : 2;  // steps of K (and of V) in shared memory
  static constexpr int Q_BYTES = CH_M * D * 2;
  static constexpr int KV_BYTES = CH_KEYS * D * 2;
  static constexpr int LIST = CH_SEGS * static_cast<int>(sizeof(ChunkSeg)) + CH_NT * static_cast<int>(sizeof(ChunkRow));
  static constexpr int USED = 1024 + 2 * Q_BYTES + 2 * STAGES * KV_BYTES + LIST + 512;
  static constexpr int SMEM = USED > TMEM_ALL_SMEM ? USED : TMEM_ALL_SMEM;  // all of the tensor memory
  static_assert(SMEM <= HEAD_SMEM_LIMIT, "shared memory");
};

struct ChunkArgs {
  AttnArgs a;        // L, B, T, the tensors, scale_log2; not its workspace
  int per_tile;      // tokens of a tile: 128 / G
  int window;        // 0: none
  int slot_rows;     // query rows of a part in the workspace
  float* part_o;     // [2 * CTAs][slot_rows][D]
  float2* part_ml;   // [2 * CTAs][slot_rows]
  ChunkCut* cuts;    // [CTAs]
};

Q3S_DEV ChunkRow chunk_row(const AttnArgs& a, int b) {
  const int o0 = a.offsets[b], o1 = a.offsets[b + 1], len = a.lengths[b];
  ChunkRow x;
  x.t0 = min(max(o0, 0), a.T);
  x.n = min(max(o1, x.t0), a.T) - x.t0;
  x.len = static_cast<int>(min(static_cast<int64_t>(max(len, 0)), static_cast<int64_t>(a.max_blocks) * a.bs));
  return x;
}
// Steps of the item of tokens [i0, i0 + m) of a row: first and count (0: its queries see nothing).
Q3S_DEV int2 chunk_steps(const ChunkArgs& c, const ChunkRow& x, int i0, int m) {
  const int L = c.a.L;
  auto step_of = [&](int p) { return p < L ? p / CH_KEYS : (L + CH_KEYS - 1) / CH_KEYS + (p - L) / CH_KEYS; };
  const int hi = L + max(x.len - x.n + i0 + m, 0) - 1;  // the last position that is seen
  if (hi < 0) return make_int2(0, 0);
  const int64_t lo = c.window ? static_cast<int64_t>(L) + x.len - x.n + i0 - c.window + 1 : 0;
  const int first = step_of(static_cast<int>(max(lo, static_cast<int64_t>(0))));
  return make_int2(first, step_of(hi) - first + 1);
}

// Where a CTA is in the list.
struct ChunkWalk {
  int b, i, h;  // row, first token in it, head: the item that starts at `at`
  int written, cut, more;
  long long at, all;
};

// Boundaries of the CTAs' ranges: CTA i has [all * i / ctas, all * (i + 1) / ctas).
struct ChunkCutting {
  long long all;
  int ctas;
  Q3S_DEV long long start(int i) const { return all * i / ctas; }
  Q3S_DEV int cta_of(long long at) const { return static_cast<int>(((at + 1) * ctas + all - 1) / all) - 1; }
};

// One query row of a segment again, key by key: what it does not see is left out
// instead of taken times p = 0, where an infinity or NaN in V would reach it.
// One warp, D / 32 dims a lane.
template <int D, bool BF16>
Q3S_DEV void chunk_row_by_key(const ChunkArgs& c, const ChunkSeg& g, int token, int gq, int own, int64_t first, int lane, float (&acc)[D / 32],
                              float& m, float& l) {
  const AttnArgs& a = c.a;
  constexpr int E = D / 32;
  auto dims = [&](const void* at, int64_t offset, float (&y)[E]) {
    const uint32_t* p = reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(at) + offset + lane * E);
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const float2 f = unpack2<BF16>(p[e / 2]);
      y[e] = f.x, y[e + 1] = f.y;
    }
  };
  float q[E];
  dims(a.q, static_cast<int64_t>(token) * a.qt + (static_cast<int64_t>(g.h) * a.G + gq) * a.qh, q);
  m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.0f;
  const int before = (a.L + CH_KEYS - 1) / CH_KEYS;
#pragma unroll 1
  for (int s = g.step0; s < g.step0 + g.steps; ++s) {
    const bool prefix = s < before;
    const int key0 = (prefix ? s : s - before) * CH_KEYS, end = min(prefix ? a.L : own, key0 + CH_KEYS);
    const int64_t base = prefix ? 0 : a.L;
    const int32_t* blocks = prefix ? a.prefix_blocks : a.table + g.b * a.table_stride;
#pragma unroll 1
    for (int j = key0; j < end; ++j) {
      if (base + j < first) continue;
      const int id = blocks[j >> a.bs_log2], place = j & (a.bs - 1);
      float k[E], v[E], x = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) k[e] = v[e] = 0.0f;
      if (static_cast<unsigned>(id) < static_cast<unsigned>(a.blocks)) {
        dims(a.k, id * a.kb + g.h * a.kh + place * a.kp, k);
        dims(a.v, id * a.vb + g.h * a.vh + place * a.vp, v);
      }
#pragma unroll
      for (int e = 0; e < E; ++e) x = fmaf(q[e], k[e], x);
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) x += __shfl_xor_sync(FULL, x, d);
      x *= a.scale_log2;
      const float nm = fmaxf(m, x), bm = nm == -INFINITY ? 0.0f : nm, w = ex2(m - bm), p = ex2(x - bm);
      m = nm;
      l = l * w + p;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = acc[e] * w + p * v[e];
    }
  }
}

// 1 / l, or what stands for it: 0 where nothing was seen, a NaN where l is one.
Q3S_DEV float chunk_inverse(float l) { return l > 0.0f ? 1.0f / l : l == l ? 0.0f : l; }
Q3S_DEV float chunk_lse(float m, float l) { return l > 0.0f ? (m + log2f(l)) * 0.69314718055994531f : l == l ? -INFINITY : l; }

// The matrix warp alternates between the two tiles as the shared-prefix kernel
// does (q3s_attn_prefix.cuh), here over the steps of one segment after another:
//   O0 += P0 V, S0 = Q0 K'^T, O1 += P1 V, S1 = Q1 K'^T,
// where K' is the next step's, of the next segment after a segment's last, so
// that a segment's start overlaps the end of the one before.  A tile's O is taken
// out by its softmax warps before they write the next segment's first P, which
// is what the next product into O waits for; Q is replaced once the
// last scores of a segment are complete.  A softmax thread owns a query row; m, l and the
// sum of the rounded p are in registers.  TMEM: S0 S1 O0 O1, 128 columns each.
//
// Masks are a range of columns a row and step (behind the query's own place, before the window, past the prefix's end); steps
// that all rows of a warp see whole skip them.  V is cleared past the end of a
// row's (or the prefix's) last step by the softmax warps of tile 0 before they hand over their first P of it;
// whole pages past the end read as zeros.
template <int D, bool BF16>
__global__ void __launch_bounds__(CH_NT, 1)
    attn_chunk_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const ChunkArgs c) {
  using Tile = ChunkTile<D>;
  constexpr int HALVES = Tile::HALVES, STAGES = Tile::STAGES;
  const AttnArgs& a = c.a;
  extern __shared__ __align__(1024) unsigned char ch_smem[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(ch_smem) + 1023) &
                                                         ~static_cast<uintptr_t>(1023));
  unsigned char* s_q = smem;
  unsigned char* s_k = s_q + 2 * Tile::Q_BYTES;
  unsigned char* s_v = s_k + STAGES * Tile::KV_BYTES;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(s_v + STAGES * Tile::KV_BYTES);
  uint64_t* q_empty = q_full + 1;
  uint64_t* k_full = q_empty + 1;
  uint64_t* k_empty = k_full + STAGES;
  uint64_t* v_full = k_empty + STAGES;
  uint64_t* v_empty = v_full + STAGES;
  uint64_t* s_full = v_empty + STAGES;  // [2] scores of a tile are in TMEM
  uint64_t* p_half = s_full + 2;        // [2] the probabilities of its first 64 keys are
  uint64_t* p_full = p_half + 2;        // [2] all are
  uint64_t* o_done = p_full + 2;        // [2] its second product is complete
  uint64_t* done = o_done + 2;          // behind a wait that gave up
  long long* s_sum = reinterpret_cast<long long*>(done + 1);  // [CH_NT / 32]
  long long* s_at = s_sum + CH_NT / 32;
  ChunkWalk* walker = reinterpret_cast<ChunkWalk*>(s_at + 1);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(walker + 1);
  int* failed = reinterpret_cast<int*>(tmem_slot + 1);
  int *s_row = failed + 1, *s_segs = s_row + 1, *s_more = s_segs + 1;
  static_assert((2 + 4 * STAGES + 8 + 1 + CH_NT / 32 + 1) * 8 + sizeof(ChunkWalk) + 5 * 4 <= 512, "room for the barriers and counts");
  ChunkSeg* s_list = reinterpret_cast<ChunkSeg*>(reinterpret_cast<unsigned char*>(q_full) + 512);
  ChunkRow* s_rows = reinterpret_cast<ChunkRow*>(s_list + CH_SEGS);  // the first CH_NT rows
  const int t = static_cast<int>(threadIdx.x), w = t >> 5, lane = t & 31;
  const int cta = static_cast<int>(blockIdx.x);
  const int pair = 2 * c.per_tile;  // tokens of an item
  const int before = (a.L + CH_KEYS - 1) / CH_KEYS;  // the prefix's steps

  grid_wait();
  grid_release();
  if (w == 8) {
    if (lane < 3) prefetch_map(lane == 0 ? &tm_q : lane == 1 ? &tm_k : &tm_v);
    if (lane == 0) {
      mbar_init(q_full, 1);
      mbar_init(q_empty, 1);
      mbar_init(done, 1);
      for (int s = 0; s < STAGES; ++s) {
        mbar_init(&k_full[s], 1);
        mbar_init(&k_empty[s], 1);
        mbar_init(&v_full[s], 1);
        mbar_init(&v_empty[s], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&s_full[i], 1);
        mbar_init(&p_half[i], 128);
        mbar_init(&p_full[i], 128);
        mbar_init(&o_done[i], 1);
      }
      *failed = 0;
      fence_mbar_init();
    }
    __syncwarp();
  }
  if (w == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }

  // ---- the list's length, and this CTA's range of it ----
  auto step_cost = [&](int m) { return m > c.per_tile ? 3 : 2; };
  auto row_cost = [&](const ChunkRow& x) {
    long long r = 0;
    for (int i0 = 0; i0 < x.n; i0 += pair) {
      const int m = min(pair, x.n - i0), steps = chunk_steps(c, x, i0, m).y;
      if (steps) r += static_cast<long long>(a.H) * (CH_START + static_cast<long long>(steps) * step_cost(m));
    }
    return r;
  };
  long long mine = 0, all = 0;  // this thread's row of the first CH_NT, all of its rows
  for (int b = t; b < a.B; b += CH_NT) {
    const ChunkRow x = chunk_row(a, b);
    const long long r = row_cost(x);
    if (b == t) {
      mine = r;
      s_rows[t] = x;
    }
    all += r;
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) all += __shfl_xor_sync(FULL, all, d);
  if (lane == 0) s_sum[w] = all;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  all = 0;
#pragma unroll
  for (int i = 0; i < CH_NT / 32; ++i) all += s_sum[i];
  // as many CTAs as every range holds the start of a step for
  const int ctas = static_cast<int>(min(static_cast<long long>(gridDim.x), max(all / CH_MAX_STEP, 1ll)));
  const bool works = all > 0 && cta < ctas;
  if (works) {  // the row in which the range starts
    const long long range0 = ChunkCutting{all, ctas}.start(cta);
    long long carry = 0;
    for (int b0 = 0; b0 < a.B && carry <= range0; b0 += CH_NT) {
      const long long r = b0 == 0 ? mine : b0 + t < a.B ? row_cost(chunk_row(a, b0 + t)) : 0;
      long long up = r;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const long long o = __shfl_up_sync(FULL, up, d);
        if (lane >= d) up += o;
      }
      __syncthreads();  // the sums before have been read
      if (lane == 31) s_sum[w] = up;
      __syncthreads();
      long long at = carry + up - r;
#pragma unroll
      for (int i = 0; i < CH_NT / 32; ++i) {
        if (i < w) at += s_sum[i];
        carry += s_sum[i];
      }
      if (at <= range0 && range0 < at + r) {
        *s_row = b0 + t;
        *s_at = at;
      }
    }
    __syncthreads();
  }
  // Thread 0 walks the list from there and writes the segments, CH_SEGS at a time
  // (where it is stands in shared memory: the registers are the softmax's).
  if (t == 0) {
    if (works) *walker = {*s_row, 0, 0, 0, 0, 1, *s_at, all};
    else c.cuts[cta].parts = 0;
  }
  auto walk = [&]() {  // thread 0
    ChunkWalk k = *walker;
    const ChunkCutting cut = {k.all, ctas};
    const long long range0 = cut.start(cta), range1 = cut.start(cta + 1);
    auto row_at = [&](int b) { return b < CH_NT ? s_rows[b] : chunk_row(a, b); };
    ChunkRow x = k.b < a.B ? row_at(k.b) : ChunkRow{0, 0, 0};
    int n = 0;
    while (k.more && n < CH_SEGS) {
      if (k.i >= x.n) {  // the next row
        if (++k.b >= a.B) {
          k.more = 0;
          break;
        }
        x = row_at(k.b);
        k.i = 0;
        continue;
      }
      const int m = min(pair, x.n - k.i), each = step_cost(m);
      const int2 steps = chunk_steps(c, x, k.i, m);
      const long long cost = steps.y ? CH_START + static_cast<long long>(steps.y) * each : 0;
      if (steps.y == 0 || (k.h == 0 && k.at + a.H * cost <= range0)) {  // nothing to see, or before the range
        k.at += a.H * cost;
        k.i += pair;
        continue;
      }
      if (k.h == 0 && k.at < range0) {
        k.h = static_cast<int>((range0 - k.at) / cost);
        k.at += k.h * cost;
      }
      if (k.at >= range1) {
        k.more = 0;
        break;
      }
      const long long start = k.at + CH_START;  // of its first step
      auto steps_before = [&](long long y) {    // that start before y
        return y <= start ? 0 : static_cast<int>(min((y - start + each - 1) / each, static_cast<long long>(steps.y)));
      };
      const int lo = steps_before(range0), hi = steps_before(range1);
      if (lo < hi) {
        ChunkSeg& g = s_list[n++];
        g.b = k.b;
        g.h = k.h;
        g.token = x.t0 + k.i;
        g.tokens = m;
        g.i_key = x.len - x.n + k.i + 1;
        g.len = x.len;
        g.step0 = steps.x + lo;
        g.steps = hi - lo;
        g.slot = lo == 0 && hi == steps.y ? -1 : 2 * cta + (k.written ? 1 : 0);
        k.written = 1;
        if (lo == 0 && hi < steps.y) {
          c.cuts[cta] = {cut.cta_of(start + static_cast<long long>(steps.y - 1) * each) - cta + 1, g.slot, cta, k.h, g.token, m};
          k.cut = 1;
        }
      }
      k.at += cost;
      if (++k.h == a.H) k.h = 0, k.i += pair;
    }
    if (!k.more && !k.cut) c.cuts[cta].parts = 0;
    *walker = k;
    *s_segs = n;
    *s_more = k.more;
  };

  // a wait that gives up marks the CTA; every role then stops at its next wait
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*reinterpret_cast<volatile int*>(failed)) return false;
    if (mbar_wait_bounded(bar, parity)) return true;
    atomicOr(failed, 1);
    return false;
  };
  const int rows = min(a.bs, CH_KEYS), pages = CH_KEYS / rows;
  int kv = 0, segs = 0;  // steps and segments so far (softmax warps: kv counts the steps of their tile)
  int cnt[2] = {0, 0};   // the matrix warp's steps of each tile
  int k_copies = 0, v_copies = 0, q_copies = 0, bad = 0;
  bool ok = true;

  for (bool again = works; again;) {
    if (t == 0) walk();
    __syncthreads();
    const int n = *s_segs;
    again = *s_more;
    if (w == 8) {
      // ---- copies: lane l copies box l of a step (a page, or 128 tokens of one) ----
      auto block_of = [&](const ChunkSeg& g, int j) {  // past the cache (it reads as zeros) where there is none
        const int s = g.step0 + j;
        const bool prefix = s < before;
        const int key = (prefix ? s : s - before) * CH_KEYS + lane * rows;
        if (lane >= pages || key >= (prefix ? a.L : g.len)) return a.blocks;
        const int32_t* ids = prefix ? a.prefix_blocks : a.table + g.b * a.table_stride;
        return ids[key >> a.bs_log2];
      };
      auto copy = [&](const CUtensorMap* map, unsigned char* ring, uint64_t* full, int h, int block) {
        const int s = kv % STAGES, place = (lane * rows) & (a.bs - 1);
        if (lane == 0) mbar_expect_tx(&full[s], Tile::KV_BYTES);
        __syncwarp();
        if (lane < pages)
          for (int x = 0; x < HALVES; ++x)
            tma_load_slice(smem_u32(ring + s * Tile::KV_BYTES + x * CH_KEYS * 128 + lane * rows * 128), map, x, place, h, block, &full[s]);
      };
      int next = n ? block_of(s_list[0], 0) : 0;
      for (int e = 0; ok && e < n; ++e) {
        const ChunkSeg g = s_list[e];
        const int tiles = g.tokens > c.per_tile ? 2 : 1;
        for (int j = 0; ok && j < g.steps; ++j) {
          const bool inside = static_cast<unsigned>(next) < static_cast<unsigned>(a.blocks);
          bad |= !inside && next != a.blocks;
          const int block = inside ? next : a.blocks;
          if (j + 1 < g.steps) next = block_of(g, j + 1);
          else if (e + 1 < n) next = block_of(s_list[e + 1], 0);
          const int s = kv % STAGES;
          const uint32_t parity = static_cast<uint32_t>(kv / STAGES - 1) & 1u;
          if (kv >= STAGES && !(ok = __all_sync(FULL, wait(&k_empty[s], parity)))) break;
          copy(&tm_k, s_k, k_full, g.h, block);
          ++k_copies;
          if (j == 0) {
            if (segs && !(ok = __all_sync(FULL, wait(q_empty, static_cast<uint32_t>(segs - 1) & 1u)))) break;
            if (lane == 0) {
              mbar_expect_tx(q_full, static_cast<uint32_t>(tiles * HALVES * c.per_tile * a.G * 128));
              for (int i = 0; i < tiles; ++i)
                for (int x = 0; x < HALVES; ++x)
                  tma_load_3d(smem_u32(s_q + i * Tile::Q_BYTES + x * CH_M * 128), &tm_q, 64 * x, g.h * a.G, g.token + i * c.per_tile, q_full);
            }
            __syncwarp();
            ++q_copies;
            ++segs;
          }
          if (kv >= STAGES && !(ok = __all_sync(FULL, wait(&v_empty[s], parity)))) break;
          copy(&tm_v, s_v, v_full, g.h, block);
          ++v_copies;
          ++kv;
        }
      }
    } else if (w == 9) {
      // ---- products --------------------------------------------------------------
      constexpr uint32_t FMT = BF16 ? 1u : 0u;
      constexpr uint32_t ID_S = (1u << 4) | (FMT << 7) | (FMT << 10) | (static_cast<uint32_t>(CH_KEYS >> 3) << 17) |
                                (static_cast<uint32_t>(CH_M >> 4) << 24);
      constexpr uint32_t ID_O = (1u << 4) | (FMT << 7) | (FMT << 10) | (1u << 16) | (static_cast<uint32_t>(D >> 3) << 17) |
                                (static_cast<uint32_t>(CH_M >> 4) << 24);  // bit 16: B's rows are the contraction
      const int kv0 = kv, segs0 = segs, cnt0[2] = {cnt[0], cnt[1]};
      if (elect_one()) {
        const uint64_t q_desc = head_smem_desc(smem_u32(s_q)), k_desc = head_smem_desc(smem_u32(s_k)), v_desc = v_smem_desc(smem_u32(s_v));
        auto scores = [&](int i, int s) {  // S_i = Q_i K^T
          const uint64_t dq = q_desc + static_cast<uint64_t>(i * (Tile::Q_BYTES >> 4)), dk = k_desc + static_cast<uint64_t>(s * (Tile::KV_BYTES >> 4));
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            constexpr int SLICE = (CH_KEYS * 128) >> 4;
            umma_f16(tmem + static_cast<uint32_t>(128 * i), dq + (k / 4) * SLICE + (k % 4) * 2, dk + (k / 4) * SLICE + (k % 4) * 2, ID_S, k != 0);
          }
          umma_commit(&s_full[i]);
        };
        // the scores of a step: its first tile waits for their operands
        auto next_scores = [&](int i, int tiles, int step, bool first, bool last) {
          const int s = step % STAGES;
          if (i == 0) {
            if (first) ok = ok && wait(q_full, static_cast<uint32_t>(segs++) & 1u);
            ok = ok && wait(&k_full[s], static_cast<uint32_t>(step / STAGES) & 1u);
            if (!ok) return;
            tc_fence_after();
          }
          scores(i, s);
          if (i == tiles - 1) {
            umma_commit(&k_empty[s]);
            if (last) umma_commit(q_empty);
          }
        };
        auto tiles_of = [&](int e) { return s_list[e].tokens > c.per_tile ? 2 : 1; };
        if (n) {
          const int tiles = tiles_of(0);
          for (int i = 0; ok && i < tiles; ++i) next_scores(i, tiles, kv, true, s_list[0].steps == 1);
        }
        for (int e = 0; ok && e < n; ++e) {
          const int steps = s_list[e].steps, tiles = tiles_of(e);
          for (int j = 0; ok && j < steps; ++j, ++kv) {
            const int s = kv % STAGES;
            const bool fresh = j + 1 == steps;  // the next step is the next segment's first
            const int following = fresh ? (e + 1 < n ? s_list[e + 1].steps : 0) : steps - j - 1;  // steps from the next on
            const int next_tiles = following == 0 ? 0 : fresh ? tiles_of(e + 1) : tiles;
            ok = wait(&v_full[s], static_cast<uint32_t>(kv / STAGES) & 1u);
            for (int i = 0; ok && i < 2; ++i) {
              if (i < tiles) {
                const uint64_t dv = v_desc + static_cast<uint64_t>(s * (Tile::KV_BYTES >> 4));
#pragma unroll
                for (int half = 0; half < 2; ++half) {  // O_i += P_i V
                  ok = ok && wait(half ? &p_full[i] : &p_half[i], static_cast<uint32_t>(cnt[i]) & 1u);
                  if (!ok) break;
                  tc_fence_after();
#pragma unroll
                  for (int q = 0; q < CH_KEYS / 32; ++q) {
                    const int k = half * (CH_KEYS / 32) + q;
                    umma_f16_ta(tmem + static_cast<uint32_t>(256 + 128 * i), tmem + static_cast<uint32_t>(128 * i + 8 * k),
                                dv + k * ((16 * 128) >> 4), ID_O, (j | k) != 0);
                  }
                }
                if (!ok) break;
                if (i == tiles - 1) umma_commit(&v_empty[s]);
                umma_commit(&o_done[i]);
                ++cnt[i];
              }
              if (i < next_tiles) next_scores(i, next_tiles, kv + 1, fresh, following == 1);
            }
          }
        }
      }
      __syncwarp();
      // the counts, for whichever lane is elected next
      kv = kv0, segs = segs0 + n, cnt[0] = cnt0[0], cnt[1] = cnt0[1];
      for (int e = 0; e < n; ++e) {
        kv += s_list[e].steps;
        cnt[0] += s_list[e].steps;
        if (s_list[e].tokens > c.per_tile) cnt[1] += s_list[e].steps;
      }
    } else {
      // ---- softmax ----------------------------------------------------------------
      const int i = w >> 2, row = (w & 3) * 32 + lane;
      const uint32_t lanes = static_cast<uint32_t>((w & 3) * 32) << 16;
      const uint32_t ts = tmem + lanes + static_cast<uint32_t>(128 * i), to = tmem + lanes + static_cast<uint32_t>(256 + 128 * i);
      for (int e = 0; ok && e < n; ++e) {
        const ChunkSeg& g = s_list[e];
        if (i > 0 && g.tokens <= c.per_tile) continue;
        const int token = i * c.per_tile + row / a.G, gq = row % a.G;
        const bool exists = row < c.per_tile * a.G && token < g.tokens;
        const bool sees = exists && (!a.slot_map || a.slot_map[g.token + token] >= 0);
        const int own = sees ? g.i_key + token : 0;  // own tokens that this query sees, and the first position
        const int64_t first = sees && c.window ? max(static_cast<int64_t>(a.L) + own - c.window, static_cast<int64_t>(0)) : 0;
        float m = -INFINITY, l = 0.0f, lr = 0.0f;  // lr: of the rounded p
        for (int j = 0; j < g.steps; ++j, ++kv) {
          const int s = g.step0 + j;
          const bool prefix = s < before;
          const int key0 = (prefix ? s : s - before) * CH_KEYS;  // of the prefix or of the row's own
          ok = __all_sync(FULL, wait(&s_full[i], static_cast<uint32_t>(kv) & 1u));
          if (!ok) break;
          tc_fence_after();
          uint32_t r[128];
          tmem_ld128(ts, r);
          // the columns that are seen: [c_lo, c_hi)
          const int c_hi = sees ? (prefix ? a.L : own) - key0 : 0;
          const int c_lo = static_cast<int>(min(max(first - key0 - (prefix ? 0 : a.L), static_cast<int64_t>(0)), static_cast<int64_t>(CH_KEYS)));
          if (__any_sync(FULL, c_hi < CH_KEYS || c_lo > 0)) {
#pragma unroll
            for (int x = 0; x < 128; ++x)
              if (x >= c_hi || x < c_lo) r[x] = 0xff800000u;
          }
          auto f = [&](int x) { return __uint_as_float(r[x]); };
          float x4[4] = {f(0), f(1), f(2), f(3)};
#pragma unroll
          for (int x = 4; x + 8 <= 128; x += 8) {
#pragma unroll
            for (int y = 0; y < 4; ++y) x4[y] = max3(x4[y], f(x + 2 * y), f(x + 2 * y + 1));
          }
#pragma unroll
          for (int y = 0; y < 4; ++y) x4[y] = fmaxf(x4[y], f(124 + y));
          const float top = max3(fmaxf(x4[0], x4[1]), x4[2], x4[3]) * a.scale_log2;
          const bool rise = top > m + PX_SLACK || (j == 0 && top > m);
          if (__any_sync(FULL, rise)) {
            const float nm = rise ? top : m;
            const float k = rise ? ex2(m - nm) : 1.0f;  // 0 from -inf
            l *= k;
            lr *= k;
            m = nm;
            if (j > 0) {
              ok = __all_sync(FULL, wait(&o_done[i], static_cast<uint32_t>(kv - 1) & 1u));
              if (!ok) break;
              tc_fence_after();
#pragma unroll 1
              for (int y = 0; y < D / 32; ++y) {
                float v[32];
                tmem_ld32(to + static_cast<uint32_t>(32 * y), v);
                uint32_t u[32];
#pragma unroll
                for (int x = 0; x < 32; ++x) u[x] = __float_as_uint(v[x] * k);
                tmem_st32(to + static_cast<uint32_t>(32 * y), u);
              }
            }
          }
          const int valid = (prefix ? a.L : g.len) - key0, end = min((valid + rows - 1) / rows * rows, CH_KEYS);
          if (i == 0 && valid < end) {  // V past the end, up to the end of its box
            const int stage = kv % STAGES;
            ok = __all_sync(FULL, wait(&v_full[stage], static_cast<uint32_t>(kv / STAGES) & 1u));
            if (!ok) break;
            for (int x = t; x < (end - valid) * 8 * HALVES; x += 128) {
              const int half = x / ((end - valid) * 8), at = x - half * (end - valid) * 8;
              *reinterpret_cast<uint4*>(s_v + stage * Tile::KV_BYTES + half * CH_KEYS * 128 + valid * 128 + at * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
          }
          const float base = m == -INFINITY ? 0.0f : m;
          const float2 sc = make_float2(a.scale_log2, a.scale_log2), nb = make_float2(-base, -base);
          float2 sum0 = make_float2(0.0f, 0.0f), sum1 = sum0, rounded0 = sum0, rounded1 = sum0;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t pk[32];
#pragma unroll
            for (int x = 0; x < 32; ++x) {
              float2 p = __ffma2_rn(make_float2(f(64 * half + 2 * x), f(64 * half + 2 * x + 1)), sc, nb);
              p.x = ex2(p.x);
              p.y = ex2(p.y);
              if (x & 1) sum1 = __fadd2_rn(sum1, p); else sum0 = __fadd2_rn(sum0, p);
              pk[x] = pack2<BF16>(p.x, p.y);
              const float2 r2 = unpack2<BF16>(pk[x]);
              if (x & 1) rounded1 = __fadd2_rn(rounded1, r2); else rounded0 = __fadd2_rn(rounded0, r2);
            }
            tmem_st32(ts + static_cast<uint32_t>(32 * half), pk);
            tc_fence_before();
            mbar_arrive(half ? &p_full[i] : &p_half[i]);
          }
          l += (sum0.x + sum1.x) + (sum0.y + sum1.y);
          lr += (rounded0.x + rounded1.x) + (rounded0.y + rounded1.y);
        }
        if (!ok) break;
        ok = __all_sync(FULL, wait(&o_done[i], static_cast<uint32_t>(kv - 1) & 1u));
        if (!ok) break;
        tc_fence_after();
        // out = O / (sum of the rounded p); a part: O times l over that sum, with m and l
        const bool whole = g.slot < 0;
        const bool some = !(l == 0.0f);  // (a NaN is some)
        const float even = lr > 0.0f ? l / lr : 1.0f, factor = whole ? even * chunk_inverse(l) : even;
        const int64_t out_at = static_cast<int64_t>(g.token + token) * a.ot + (static_cast<int64_t>(g.h) * a.G + gq) * a.oh;
        const int64_t part_at = static_cast<int64_t>(max(g.slot, 0)) * c.slot_rows + i * c.per_tile * a.G + row;
        float odd = 0.0f;  // a NaN where a value is not finite
#pragma unroll 1
        for (int y = 0; y < D / 32; ++y) {
          float v[32];
          tmem_ld32(to + static_cast<uint32_t>(32 * y), v);
#pragma unroll
          for (int x = 0; x < 32; ++x) {
            odd = fmaf(v[x], 0.0f, odd);
            v[x] = some ? v[x] * factor : 0.0f;
          }
          if (exists) {
            if (whole) {
              uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + out_at + 32 * y);
#pragma unroll
              for (int x = 0; x < 4; ++x)
                dst[x] = make_uint4(pack2<BF16>(v[8 * x], v[8 * x + 1]), pack2<BF16>(v[8 * x + 2], v[8 * x + 3]),
                                    pack2<BF16>(v[8 * x + 4], v[8 * x + 5]), pack2<BF16>(v[8 * x + 6], v[8 * x + 7]));
            } else {
              float4* dst = reinterpret_cast<float4*>(c.part_o + part_at * D + 32 * y);
#pragma unroll
              for (int x = 0; x < 8; ++x) dst[x] = make_float4(v[4 * x], v[4 * x + 1], v[4 * x + 2], v[4 * x + 3]);
            }
          }
        }
        tc_fence_before();  // O has been read: the next P of this tile (its barrier) lets the next product into it start
        if (exists) {
          if (!whole) c.part_ml[part_at] = make_float2(m, l);
          else if (a.lse) a.lse[static_cast<int64_t>(g.token + token) * a.Hq + g.h * a.G + gq] = chunk_lse(m, l);
        }
        // sums that are not finite though the scores are: V holds an infinity or a NaN
        unsigned redo = __ballot_sync(FULL, sees && odd != odd && l > 0.0f && l < INFINITY);
        while (redo) {
          const int src = __ffs(redo) - 1;
          redo &= redo - 1;
          const int tk = __shfl_sync(FULL, token, src), q = __shfl_sync(FULL, gq, src), ow = __shfl_sync(FULL, own, src);
          const int64_t fi = __shfl_sync(FULL, first, src), at = __shfl_sync(FULL, part_at, src), oat = __shfl_sync(FULL, out_at, src);
          constexpr int E = D / 32;
          float acc[E], km, kl;
          chunk_row_by_key<D, BF16>(c, g, g.token + tk, q, ow, fi, lane, acc, km, kl);
          __syncwarp();  // its writes come after those above
          if (whole) {
            const float inv = chunk_inverse(kl);
            uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + oat + lane * E);
#pragma unroll
            for (int x = 0; x < E; x += 2) dst[x / 2] = pack2<BF16>(acc[x] * inv, acc[x + 1] * inv);
          } else {
#pragma unroll
            for (int x = 0; x < E; ++x) c.part_o[at * D + lane * E + x] = acc[x];
            if (lane == 0) c.part_ml[at] = make_float2(km, kl);
          }
        }
      }
    }
    __syncthreads();  // the segments have been taken, the next ones may be listed
    if (*reinterpret_cast<volatile int*>(failed)) break;
  }

  if (w == 8) {
    if (bad && a.error_word) atomicOr(a.error_word, Q3S_DECERR_BLOCK_ID);
    // no copy may be in flight when the CTA leaves: wait for each stage's last one
    if (lane == 0) {
      if (q_copies) (void)mbar_wait_bounded(q_full, static_cast<uint32_t>(q_copies - 1) & 1u);
      for (int i = max(0, k_copies - STAGES); i < k_copies; ++i)
        (void)mbar_wait_bounded(&k_full[i % STAGES], static_cast<uint32_t>(i / STAGES) & 1u);
      for (int i = max(0, v_copies - STAGES); i < v_copies; ++i)
        (void)mbar_wait_bounded(&v_full[i % STAGES], static_cast<uint32_t>(i / STAGES) & 1u);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (w == 9) {
    tc_fence_after();
    if (*failed) {  // products may still be running: a commit behind them (bounded) before the columns go
      if (elect_one()) {
        umma_commit(done);
        (void)mbar_wait_bounded(done, 0);
      }
      __syncwarp();
    }
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
  if (t == 0 && *failed && a.error_word) atomicOr(a.error_word, Q3S_DECERR_WAIT);
}

// Joins the parts of the items that were cut, a warp a query row; blocks behind
// those write 0 and -inf for the tokens that no item has (of no row, or that see nothing).
template <int D, bool BF16>
__global__ void __launch_bounds__(CH_JOIN_NT) attn_chunk_join_kernel(const ChunkArgs c, int join_blocks, int blocks_each) {
  constexpr int E = D / 32, AHEAD = 4;
  const AttnArgs& a = c.a;
  const int t = static_cast<int>(threadIdx.x), w = t >> 5, lane = t & 31, block = static_cast<int>(blockIdx.x);
  grid_wait();
  grid_release();
  if (block < join_blocks) {
    const ChunkCut k = c.cuts[block / blocks_each];
    if (k.parts == 0) return;
    const int rows = k.tokens * a.G, row0 = (block % blocks_each) * CH_JOIN_ROWS;
    for (int r = row0 + w; r < min(rows, row0 + CH_JOIN_ROWS); r += CH_JOIN_NT / 32) {
      float acc[E], m = -INFINITY, l = 0.0f;
#pragma unroll
      for (int x = 0; x < E; ++x) acc[x] = 0.0f;
      for (int i = 0; i < k.parts; i += AHEAD) {
        float y[AHEAD][E];
        float2 ml[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
          ml[j] = make_float2(-INFINITY, 0.0f);
          if (i + j < k.parts) {
            const int64_t at = static_cast<int64_t>(i + j == 0 ? k.slot : 2 * (k.cta + i + j)) * c.slot_rows + r;
            ml[j] = c.part_ml[at];
            const float* src = c.part_o + at * D + lane * E;
            if constexpr (E == 4) {
              const float4 f = *reinterpret_cast<const float4*>(src);
              y[j][0] = f.x, y[j][1] = f.y, y[j][2] = f.z, y[j][3] = f.w;
            } else {
              const float2 f = *reinterpret_cast<const float2*>(src);
              y[j][0] = f.x, y[j][1] = f.y;
            }
          }
        }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
          if (i + j >= k.parts) break;
          const float nm = fmaxf(m, ml[j].x), base = nm == -INFINITY ? 0.0f : nm;
          const float wm = ex2(m - base), wp = ex2(ml[j].x - base);
          m = nm;
          l = l * wm + wp * ml[j].y;
#pragma unroll
          for (int x = 0; x < E; ++x) acc[x] = acc[x] * wm + wp * y[j][x];
        }
      }
      const int token = k.token + r / a.G, head = k.h * a.G + r % a.G;
      const float inv = chunk_inverse(l);
      uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + token * a.ot + head * a.oh + lane * E);
#pragma unroll
      for (int x = 0; x < E; x += 2) dst[x / 2] = pack2<BF16>(acc[x] * inv, acc[x + 1] * inv);
      if (a.lse && lane == 0) a.lse[static_cast<int64_t>(token) * a.Hq + head] = chunk_lse(m, l);
    }
    return;
  }
  const int token = (block - join_blocks) * CH_JOIN_NT + t;
  bool none = false;
  if (token < a.T) {
    none = true;
    if (a.B > 0) {
      int b = 0, end = a.B;  // offsets[b] <= token < offsets[end], if there is such a row
      while (end - b > 1) {
        const int mid = (b + end) >> 1;
        if (a.offsets[mid] <= token) b = mid; else end = mid;
      }
      const ChunkRow x = chunk_row(a, b);
      if (token >= x.t0 && token < x.t0 + x.n) {
        const int i0 = (token - x.t0) / (2 * c.per_tile) * (2 * c.per_tile);
        none = chunk_steps(c, x, i0, min(2 * c.per_tile, x.n - i0)).y == 0;
      }
    }
  }
  for (unsigned which = __ballot_sync(FULL, none); which; which &= which - 1) {
    const int64_t tk = token - lane + __ffs(which) - 1;
    for (int x = lane; x < a.Hq * (D / 8); x += 32)
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + tk * a.ot + x / (D / 8) * a.oh + x % (D / 8) * 8) = make_uint4(0, 0, 0, 0);
    if (a.lse)
      for (int x = lane; x < a.Hq; x += 32) a.lse[tk * a.Hq + x] = -INFINITY;
  }
}

}  // namespace q3s
