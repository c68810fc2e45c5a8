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
//
// Measured on the device: 2 rows of 4096 tokens behind up to 3650 keys, 16 and 8 heads of 128, 239 us (950 TFLOP/s;
// 273 us in a long run under the power limit); 13 rows of up to 700 tokens in a window of 512, 16 and 4 heads of 64,
// 50 us; 48 rows of up to 9 tokens and 1533 keys, 32 and 8 heads of 128, 60 us at first (54 by the other kernels).
// A long row is bound by the softmax and its hand-overs: two units of 64 keys take 2100 clocks, of which the tensor
// cores run 1300.  Short rows are bound by what each range and item begins and ends with: 7 us until the first scores
// (lengths, list, loads), 3 us from an item's last unit to the next one's first, and the join.
#pragma once

#include <cuda.h>

#include "q3s_attn.cuh"
#include "q3s_attn_prefix.cuh"
#include "q3s_head.cuh"

namespace q3s {

constexpr int CH_M = PX_M, CH_KEYS = PX_KEYS;
constexpr int CH_NT = 384;      // two softmax warpgroups, and one with the copy warp and three matrix warps
constexpr int CH_SEGS = 64;     // segments of a CTA's range that are listed at a time
// Registers a thread: a softmax thread holds a unit's 64 scores of its row and their probabilities.  Launched with 168 a
// thread, which is what the shares add up to.
constexpr int CH_REGS_SOFTMAX = 184, CH_REGS_OTHER = 136;
static_assert(2 * CH_REGS_SOFTMAX + CH_REGS_OTHER <= 3 * 168, "what the CTA is launched with");
constexpr int CH_START = 2;     // cost of an item's start and end, in steps (2 rows of 4096 tokens: 0.7 261 us, 2 248, 4 251, 8 264)
constexpr int CH_JOIN_NT = 256, CH_JOIN_ROWS = 32;  // threads and query rows of a CTA of the joining kernel

constexpr int CH_UNSEEN = -0x7fffffff - 1;  // in place of how many own tokens a query sees: there is none, or it sees nothing

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
  static constexpr int KEYS = 64;                  // keys of a unit
  static constexpr int PIECES = CH_KEYS / KEYS;    // units that a step's keys are cut into
  static_assert(PIECES == 2, "each softmax warpgroup has a unit of every step");
  static constexpr int BUFFERS = D == 64 ? 6 : 4;  // places for scores in TMEM
  static_assert(BUFFERS * KEYS + 2 * D == 512, "columns");
  static constexpr int Q_BYTES = CH_M * D * 2;
  static constexpr int KV_BYTES = CH_KEYS * D * 2;
  static constexpr int LIST = CH_SEGS * static_cast<int>(sizeof(ChunkSeg)) + CH_NT * static_cast<int>(sizeof(ChunkRow) + 8) + CH_M * 12;
  static constexpr int USED = 1024 + 2 * Q_BYTES + 2 * STAGES * KV_BYTES + LIST + 512;
  static constexpr int SMEM = USED > TMEM_ALL_SMEM ? USED : TMEM_ALL_SMEM;  // all of the tensor memory
  static_assert(SMEM <= HEAD_SMEM_LIMIT, "shared memory");
};

struct ChunkArgs {
  AttnArgs a;        // L, B, T, the tensors, scale_log2; not its workspace
  int per_tile;      // tokens of a tile: 128 / G
  int window;        // 0: none
  int slot_rows;     // query rows of a part in the workspace
  float* part_o;     // [2 * CTAs][D / 4][slot_rows][4]: neighbouring rows, which are neighbouring threads', side by side
                     // (a store takes a clock for each line it touches: row after row, a part's took 3 to 4 us)
  float2* part_ml;   // [2 * CTAs][slot_rows]
  ChunkCut* cuts;    // [CTAs]
};

Q3S_HOST_DEV ChunkRow chunk_row(const AttnArgs& a, int b) {
  const int o0 = a.offsets[b], o1 = a.offsets[b + 1], len = a.lengths[b];
  ChunkRow x;
  x.t0 = min(max(o0, 0), a.T);
  x.n = min(max(o1, x.t0), a.T) - x.t0;
  x.len = static_cast<int>(min(static_cast<int64_t>(max(len, 0)), static_cast<int64_t>(a.max_blocks) * a.bs));
  return x;
}
// Steps of the item of tokens [i0, i0 + m) of a row: first and count (0: its queries see nothing).
Q3S_HOST_DEV int2 chunk_steps(const ChunkArgs& c, const ChunkRow& x, int i0, int m) {
  const int L = c.a.L;
  auto step_of = [&](int p) {  // p >= 0
    const uint32_t own = static_cast<uint32_t>(p - L);
    return static_cast<int>(p < L ? static_cast<uint32_t>(p) / CH_KEYS : static_cast<uint32_t>(L + CH_KEYS - 1) / CH_KEYS + own / CH_KEYS);
  };
  const int hi = L + max(x.len - x.n + i0 + m, 0) - 1;  // the last position that is seen
  if (hi < 0) return make_int2(0, 0);
  const int64_t lo = c.window ? static_cast<int64_t>(L) + x.len - x.n + i0 - c.window + 1 : 0;
  const int first = step_of(static_cast<int>(max(lo, static_cast<int64_t>(0))));
  return make_int2(first, step_of(hi) - first + 1);
}

// Where a CTA is in the list.
struct ChunkWalk {
  int b, item;  // row, item in it (token pair times heads, and head), or -1: at the row's start
  int written, cut, more;
  int ctas;
  long long at, all;  // where that item (the row) starts; the list's length, for `ctas` CTAs
};

// Boundaries of the CTAs' ranges: CTA i has [all * i / ctas, all * (i + 1) / ctas).
struct ChunkCutting {
  long long all;
  int ctas;
  Q3S_HOST_DEV long long start(int i) const { return div_nonneg(all * i, ctas); }
  Q3S_HOST_DEV int cta_of(long long at) const { return static_cast<int>(div_nonneg((at + 1) * ctas + all - 1, all)) - 1; }
};

// Of tokens [i0, i0 + an item's) of a row, for one head; 0: nothing is seen.
Q3S_HOST_DEV long long chunk_item_cost(const ChunkArgs& c, const ChunkRow& x, int i0) {
  const int steps = chunk_steps(c, x, i0, min(2 * c.per_tile, x.n - i0)).y;
  return steps ? CH_START + static_cast<long long>(steps) : 0ll;
}

// The lanes of a warp as chunk_walk takes them (on the host, a test's).
struct ChunkLanes {
  int lane;
  template <typename T>
  Q3S_DEV T shfl(T x, int src) const { return __shfl_sync(FULL, x, src); }
  Q3S_DEV long long scan(long long up) const {  // of the lanes up to this one
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long o = __shfl_up_sync(FULL, up, d);
      if (lane >= d) up += o;
    }
    return up;
  }
  Q3S_DEV unsigned ballot(bool x) const { return __ballot_sync(FULL, x); }
  Q3S_DEV void sync() const { __syncwarp(); }
  Q3S_DEV static int first(unsigned x) { return __ffs(x) - 1; }
  Q3S_DEV static int count(unsigned x) { return __popc(x); }
};

// Lists a CTA's next segments, up to CH_SEGS of them: a warp, 32 items at once, a lane each.  After every call c.cuts[cta]
// says which cut item starts in the segments so far, or that none does (a CTA that gives up lists no more).
#pragma nv_exec_check_disable
template <typename Lanes>
Q3S_HOST_DEV void chunk_walk(const ChunkArgs& c, int cta, const ChunkRow* rows, ChunkWalk* walker, int* segs, ChunkSeg* list, const Lanes& l) {
  const AttnArgs& a = c.a;
  const int pair = 2 * c.per_tile, lane = l.lane;
  ChunkWalk k = *walker;
  l.sync();
  const ChunkCutting cut = {k.all, k.ctas};
  const long long range0 = cut.start(cta), range1 = cut.start(cta + 1);
  int n = 0;
  while (k.more && n + 32 <= CH_SEGS) {
    if (k.b >= a.B) {
      k.more = 0;
      break;
    }
    const ChunkRow x = k.b < CH_NT ? rows[k.b] : chunk_row(a, k.b);
    if (x.n == 0) {  // on to the next row that has tokens, 32 at once (row by row 0.45 us each: 255 idle rows behind one of 300 tokens 141 us, so 31)
      const int b = k.b + lane;
      const unsigned next = l.ballot(b < a.B && (b < CH_NT ? rows[b] : chunk_row(a, b)).n > 0);
      k.b += next ? l.first(next) : 32;
      continue;
    }
    const int pairs = (x.n + pair - 1) / pair;
    const long long items = static_cast<long long>(pairs) * a.H;
    if (k.item < 0) {  // the range starts in this row: skip to the tokens where it does
      int p0 = 0;
      for (; p0 < pairs; p0 += 32) {
        const long long cost = p0 + lane < pairs ? chunk_item_cost(c, x, (p0 + lane) * pair) * a.H : 0;
        const long long up = l.scan(cost);
        const unsigned past = l.ballot(k.at + up > range0);
        if (past) {
          const int f = l.first(past);
          p0 += f;
          k.at += l.shfl(up - cost, f);
          break;
        }
        k.at += l.shfl(up, 31);
      }
      k.item = p0 * a.H;
    }
    const int item = k.item + lane, p = item / a.H, h = item - p * a.H;
    const int i0 = p * pair, m = min(pair, x.n - i0);
    int2 steps = make_int2(0, 0);
    if (item < items) steps = chunk_steps(c, x, i0, m);
    const long long cost = steps.y ? CH_START + static_cast<long long>(steps.y) : 0;
    const long long up = l.scan(cost), start = k.at + up - cost;
    auto steps_before = [&](long long y) {  // that start before y
      return static_cast<int>(min(max(y - start - CH_START, 0ll), static_cast<long long>(steps.y)));
    };
    const int lo = steps_before(range0), hi = steps_before(range1);
    const unsigned live = l.ballot(lo < hi);
    const bool whole = lo == 0 && hi == steps.y;
    const int rank = l.count(live & ((1u << lane) - 1u));
    if (lo < hi) {
      const int slot = whole ? -1 : 2 * cta + (k.written + rank > 0 ? 1 : 0);
      list[n + rank] = {k.b, h, x.t0 + i0, m, x.len - x.n + i0 + 1, x.len, steps.x + lo, hi - lo, slot};
      if (lo == 0 && !whole)
        c.cuts[cta] = {cut.cta_of(start + CH_START + steps.y - 1) - cta + 1, slot, cta, h, x.t0 + i0, m};
    }
    k.cut |= l.ballot(lo < hi && lo == 0 && !whole) != 0;
    k.written += l.count(live);
    n += l.count(live);
    k.at += l.shfl(up, 31);
    if (k.at >= range1) k.more = 0;  // no later item starts before
    k.item += 32;
    if (k.item >= items) ++k.b, k.item = 0;
  }
  if (!k.cut && lane == 0) c.cuts[cta].parts = 0;
  l.sync();
  if (lane == 0) {
    *walker = k;
    *segs = n;
  }
}

// Products and commits of one lane of a converged warp, under a predicate and not a branch: their operands are
// then computed once for the warp (in a branch each product took three times as many issue slots).
Q3S_DEV void umma_ss_if(uint32_t leader, uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %0, 0;\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%1], %2, %3, %4, p;\n}" ::"r"(leader),
      "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}
Q3S_DEV void umma_ts_if(uint32_t leader, uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %0, 0;\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%1], [%2], %3, %4, p;\n}" ::"r"(leader),
      "r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate));
}
Q3S_DEV void umma_commit_if(uint32_t leader, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %0, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n}" ::"r"(leader),
      "r"(smem_u32(bar))
      : "memory");
}

// s += the two 16-bit values of p, each to its own sum (one instruction a value; unpacked first they were three a pair).
template <bool BF16>
Q3S_DEV void add_rounded(float2& s, uint32_t p) {
  if constexpr (BF16)
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tadd.f32.bf16 %0, l, %0;\n\tadd.f32.bf16 %1, h, %1;\n}" : "+f"(s.x), "+f"(s.y) : "r"(p));
  else
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tadd.f32.f16 %0, l, %0;\n\tadd.f32.f16 %1, h, %1;\n}" : "+f"(s.x), "+f"(s.y) : "r"(p));
}

// 16 consecutive columns of this thread's TMEM lane; a store is complete after tmem_st_wait.
Q3S_DEV void tmem_ld16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}
Q3S_DEV void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), "r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
      "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
Q3S_DEV void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

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

// The two softmax warpgroups take turns: unit u of the CTA's work, 128 query rows
// against half of a step's keys, is that of warpgroup u % 2.  With two tiles of query rows
// each has one; with one tile (a few drafts) the two share its keys in turn, and the one that began joins the
// other's sums to its own at the end.  Scores have BUFFERS places in TMEM, which the probabilities take over
// (16-bit, the second product's A operand), so that the scores of up to BUFFERS units are on their way or waiting:
//   O(u) += P(u) V, then S(u + BUFFERS) = Q K^T into the place that this frees,
// over the segments without a pause.  (With one place of 128 keys a warpgroup, its softmax waited for two products
// at each step: 2 rows of 4096 tokens took 252 us, with these 244.)  A warpgroup's O, D more columns each, is taken out before it hands
// over the next segment's first P, which is what the next product into O waits for, and the two tiles of Q are a ring.
// A softmax thread owns a query row; m, l and the sum of the rounded p (q3s_attn_prefix.cuh says why) are in
// registers.  It takes its exponentials with the maximum so far while it looks for the unit's own; where a score
// rises above that by more than 8, which after a segment's first unit is rare, O is rescaled and the unit taken again.
//
// Masks are a range of columns a row and unit (behind the query's own place,
// before the window, past the prefix's end), applied by 32 columns that some row of the
// warp does not see whole.  V is cleared past the end of a row's (or the prefix's)
// last step by the softmax warps that hand over its first P; whole pages past the end read as zeros.
template <int D, bool BF16>
__global__ void __launch_bounds__(CH_NT, 1)
    attn_chunk_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const ChunkArgs c) {
  using Tile = ChunkTile<D>;
  constexpr int HALVES = Tile::HALVES, STAGES = Tile::STAGES, KEYS = Tile::KEYS, PIECES = Tile::PIECES, BUFFERS = Tile::BUFFERS;
  const AttnArgs& a = c.a;
  extern __shared__ __align__(1024) unsigned char ch_smem[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(ch_smem) + 1023) &
                                                         ~static_cast<uintptr_t>(1023));
  unsigned char* s_q = smem;
  unsigned char* s_k = s_q + 2 * Tile::Q_BYTES;
  unsigned char* s_v = s_k + STAGES * Tile::KV_BYTES;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(s_v + STAGES * Tile::KV_BYTES);  // [2]
  uint64_t* q_empty = q_full + 2;                                                 // [2]
  uint64_t* k_full = q_empty + 2;
  uint64_t* k_empty = k_full + STAGES;
  uint64_t* v_full = k_empty + STAGES;
  uint64_t* v_empty = v_full + STAGES;
  uint64_t* s_full = v_empty + STAGES;  // [BUFFERS] a unit's scores are in TMEM
  uint64_t* p_full = s_full + BUFFERS;  // [BUFFERS] its probabilities are
  uint64_t* o_done = p_full + BUFFERS;  // [BUFFERS] its second product is complete
  uint64_t* given = o_done + BUFFERS;         // a shared tile's second sums may be read, and have been
  uint64_t* taken = given + 1;
  uint64_t* done = taken + 1;           // behind a wait that gave up
  long long* s_sum = reinterpret_cast<long long*>(done + 1);  // [CH_NT / 32]
  ChunkWalk* walker = reinterpret_cast<ChunkWalk*>(s_sum + CH_NT / 32);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(walker + 1);
  int* failed = reinterpret_cast<int*>(tmem_slot + 1);
  int* s_segs = failed + 1;
  static_assert((4 + 4 * STAGES + 3 * BUFFERS + 3 + CH_NT / 32) * 8 + sizeof(ChunkWalk) + 3 * 4 <= 512, "room for the barriers and counts");
  ChunkSeg* s_list = reinterpret_cast<ChunkSeg*>(reinterpret_cast<unsigned char*>(q_full) + 512);
  ChunkRow* s_rows = reinterpret_cast<ChunkRow*>(s_list + CH_SEGS);  // the first CH_NT rows
  long long* s_cost = reinterpret_cast<long long*>(s_rows + CH_NT);  // theirs
  float* s_ml = reinterpret_cast<float*>(s_cost + CH_NT);            // [128][3] m, l and the sum of the rounded p of a shared tile's second sums
  const int t = static_cast<int>(threadIdx.x), w = t >> 5, lane = t & 31;
  const int cta = static_cast<int>(blockIdx.x);
  const int pair = 2 * c.per_tile;  // tokens of an item
  const int before = (a.L + CH_KEYS - 1) / CH_KEYS;  // the prefix's steps

  grid_wait();
  grid_release();
  if (w == 0) {
    if (lane < 3) prefetch_map(lane == 0 ? &tm_q : lane == 1 ? &tm_k : &tm_v);
    if (lane == 0) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(&q_full[i], 1);
        mbar_init(&q_empty[i], 2);
      }
      for (int i = 0; i < BUFFERS; ++i) {
        mbar_init(&s_full[i], 1);
        mbar_init(&p_full[i], 128);
        mbar_init(&o_done[i], 1);
      }
      for (int s = 0; s < STAGES; ++s) {
        mbar_init(&k_full[s], 1);
        mbar_init(&k_empty[s], 2);
        mbar_init(&v_full[s], 1);
        mbar_init(&v_empty[s], 1);
      }
      mbar_init(given, 128);
      mbar_init(taken, 128);
      mbar_init(done, 3);
      *failed = 0;
      fence_mbar_init();
    }
    __syncwarp();
  }
  if (w == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }

  // ---- the list's length, and this CTA's range of it ----
  const ChunkLanes lanes_of_warp{lane};
  // a row's cost; a whole warp calls (a row of many items is its 32 lanes' work)
  auto row_cost = [&](const ChunkRow& x) {
    long long r = 0;
    const bool large = x.n > 4 * pair;
    for (int i0 = 0; i0 < x.n && !large; i0 += pair) r += chunk_item_cost(c, x, i0);
    for (unsigned rest = __ballot_sync(FULL, large); rest; rest &= rest - 1) {
      const int src = __ffs(rest) - 1;
      const ChunkRow y = {0, __shfl_sync(FULL, x.n, src), __shfl_sync(FULL, x.len, src)};
      long long sum = 0;
      for (int64_t i0 = static_cast<int64_t>(lane) * pair; i0 < y.n; i0 += 32 * pair) sum += chunk_item_cost(c, y, static_cast<int>(i0));
#pragma unroll
      for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(FULL, sum, d);
      if (lane == src) r = sum;
    }
    return r * a.H;
  };
  long long all = 0;
  bool bad_length = false;
  const int turn_row = lane * (CH_NT / 32) + w;  // neighbouring rows to different warps (13 rows of one warp, one after another: about 2 us)
  for (int b0 = 0; b0 < a.B; b0 += CH_NT) {
    const ChunkRow x = b0 + turn_row < a.B ? chunk_row(a, b0 + turn_row) : ChunkRow{0, 0, 0};
    const long long r = row_cost(x);
    if (cta == 0 && b0 + turn_row < a.B) {  // what was cut
      const int b = b0 + turn_row;
      bad_length |= a.lengths[b] != x.len || a.offsets[b] != x.t0 || a.offsets[b + 1] != x.t0 + x.n;
    }
    if (b0 == 0) {
      s_cost[turn_row] = r;
      s_rows[turn_row] = x;
    }
    all += r;
  }
  if (bad_length && a.error_word) atomicOr(a.error_word, Q3S_DECERR_LENGTHS);
  {
    const long long up = lanes_of_warp.scan(all);
    if (lane == 31) s_sum[w] = up;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  all = 0;
#pragma unroll
  for (int i = 0; i < CH_NT / 32; ++i) all += s_sum[i];
  // (a range within an item's steps holds at least one)
  const int ctas = static_cast<int>(min(static_cast<long long>(gridDim.x), max(all, 1ll)));
  const bool works = all > 0 && cta < ctas;
  if (works) {  // the row in which the range starts
    const long long range0 = ChunkCutting{all, ctas}.start(cta);
    long long carry = 0;
    for (int b0 = 0; b0 < a.B && carry <= range0; b0 += CH_NT) {
      long long r = s_cost[t];  // in order
      if (b0) r = row_cost(b0 + t < a.B ? chunk_row(a, b0 + t) : ChunkRow{0, 0, 0});
      const long long up = lanes_of_warp.scan(r);
      __syncthreads();
      if (lane == 31) s_sum[w] = up;
      __syncthreads();
      long long at = carry + up - r;
#pragma unroll
      for (int i = 0; i < CH_NT / 32; ++i) {
        if (i < w) at += s_sum[i];
        carry += s_sum[i];
      }
      if (at <= range0 && range0 < at + r) *walker = {b0 + t, -1, 0, 0, 1, ctas, at, all};
    }
  } else if (t == 0) {
    c.cuts[cta].parts = 0;
  }
  __syncthreads();

  // a wait that gives up marks the CTA; every role then stops at its next wait
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*reinterpret_cast<volatile int*>(failed)) return false;
    if (mbar_wait_bounded(bar, parity)) return true;
    atomicOr(failed, 1);
    return false;
  };
  int kv = 0, units = 0, tiles_q = 0;  // steps, units and tiles of Q so far
  bool ok = true;
  auto tiles_of = [&](const ChunkSeg& g) { return g.tokens > c.per_tile ? 2 : 1; };

  // Each role with a loop of its own over the batches of segments, so that it has its own number of registers.
  if (w >= 4) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(CH_REGS_SOFTMAX));
    int shared = 0;        // tiles so far whose keys the two warpgroups shared
    bool pending = false;  // the sums given for the last of them must have been taken before the next product into them
    for (bool again = works; again;) {
      __syncthreads();  // the segments are listed
      const int n = *s_segs;
      again = walker->more != 0;
      // ---- softmax ----------------------------------------------------------------
      const int i = (w >> 2) - 1, row = (w & 3) * 32 + lane;
      const uint32_t lanes = static_cast<uint32_t>((w & 3) * 32) << 16;
      const uint32_t ts = tmem + lanes, to = ts + static_cast<uint32_t>(BUFFERS * KEYS + D * i);
      for (int e = 0; ok && e < n; ++e) {
        const ChunkSeg& g = s_list[e];
        const bool alone = tiles_of(g) == 2;  // with its tile
        const int turn = (i - units) & 1;     // this warpgroup's first unit in the segment
        const int tile = alone ? turn : 0, stage0 = kv, end = g.steps * PIECES * (alone ? 2 : 1);  // steps before the segment; its units
        int buffer = (units + turn) % BUFFERS;
        uint32_t parity = static_cast<uint32_t>((units + turn) / BUFFERS) & 1u;
        units += end;
        kv += g.steps;
        if (turn >= end) continue;
        int last_buffer = buffer;
        uint32_t last_parity = parity;
        float m = -INFINITY, l = 0.0f, lr = 0.0f;  // lr: of the rounded p
        // Own tokens that this row's query sees, and the first position.  A row without a query, or whose query sees
        // nothing, goes along: it is told apart at the end.
        int own = CH_UNSEEN, from = 0;
        {
          const int token = tile * c.per_tile + row / a.G;
          if (row < c.per_tile * a.G && token < g.tokens && (!a.slot_map || a.slot_map[g.token + token] >= 0)) {
            own = g.i_key + token;
            if (c.window) from = static_cast<int>(max(static_cast<int64_t>(a.L) + own - c.window, static_cast<int64_t>(0)));
          }
        }
        // The pieces that all rows of the warp see whole: [full0, full1) of the prefix, [full2, full3) of the row's own.
        int full0, full1, full2, full3;
        {
          const int least = __reduce_min_sync(FULL, own == CH_UNSEEN ? 0x7fffffff : own), most = __reduce_max_sync(FULL, from);
          const int own0 = (before - g.step0) * PIECES;
          full0 = (most + KEYS - 1) / KEYS - g.step0 * PIECES;
          full1 = a.L / KEYS - g.step0 * PIECES;
          full2 = own0 + (max(most - a.L, 0) + KEYS - 1) / KEYS;
          full3 = own0 + min(max(least, 0), g.len) / KEYS;
        }
        for (int x = turn; x < end; x += 2) {
          const int piece = alone ? x >> 1 : x;
          const bool whole_piece = (piece >= full0 && piece < full1) || (piece >= full2 && piece < full3);
          int c_hi = KEYS, c_lo = 0;  // the columns that are seen: [c_lo, c_hi)
          if (!whole_piece) {
            const int step = g.step0 + piece / PIECES;
            const bool prefix = step < before;
            const int key0 = (prefix ? step : step - before) * CH_KEYS + piece % PIECES * KEYS;  // of the prefix or of the row's own
            c_hi = min(max((prefix ? a.L : own == CH_UNSEEN ? g.len : own) - key0, 0), KEYS);
            c_lo = min(max(from - key0 - (prefix ? 0 : a.L), 0), KEYS);
            if (tile == 0) {
              // of the step's keys: behind the last one, up to the end of its box, in this piece
              const int rows = min(a.bs, CH_KEYS), first = piece % PIECES * KEYS, valid = (prefix ? a.L : g.len) - key0 + first;
              const int clear = max(valid, first), last = min(min((valid + rows - 1) & ~(rows - 1), CH_KEYS), first + KEYS);
              if (clear < last) {
                const int kv_step = stage0 + piece / PIECES, stage = kv_step % STAGES;
                ok = __all_sync(FULL, wait(&v_full[stage], static_cast<uint32_t>(kv_step / STAGES) & 1u));
                if (!ok) break;
                for (int y = row; y < (last - clear) * 8 * HALVES; y += 128) {
                  const int half = HALVES == 1 || y < (last - clear) * 8 ? 0 : 1, at = y - half * (last - clear) * 8;
                  *reinterpret_cast<uint4*>(s_v + stage * Tile::KV_BYTES + half * CH_KEYS * 128 + clear * 128 + at * 16) =
                      make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async_smem();
              }
            }
          }
          ok = __all_sync(FULL, wait(&s_full[buffer], parity));
          if (!ok) break;
          tc_fence_after();
          const uint32_t place = ts + static_cast<uint32_t>(KEYS * buffer);
          uint32_t r[KEYS];
          tmem_ld64(place, r);
          if (!whole_piece) {
#pragma unroll
            for (int y = 0; y < KEYS / 32; ++y) {
              const int lo = min(max(c_lo - 32 * y, 0), 32), hi = min(max(c_hi - 32 * y, 0), 32);
              const uint32_t seen = (hi == 32 ? 0xffffffffu : (1u << hi) - 1u) & (lo == 32 ? 0u : 0xffffffffu << lo);
#pragma unroll
              for (int z = 0; z < 32; ++z) r[32 * y + z] = seen & (1u << z) ? r[32 * y + z] : 0xff800000u;
            }
          }
          auto f = [&](int z) { return __uint_as_float(r[z]); };
          float x4[4] = {f(0), f(1), f(2), f(3)};
#pragma unroll
          for (int z = 4; z + 8 <= KEYS; z += 8) {
#pragma unroll
            for (int y = 0; y < 4; ++y) x4[y] = max3(x4[y], f(z + 2 * y), f(z + 2 * y + 1));
          }
#pragma unroll
          for (int y = 0; y < 4; ++y) x4[y] = fmaxf(x4[y], f(KEYS - 4 + y));
          const float top = max3(fmaxf(x4[0], x4[1]), x4[2], x4[3]) * a.scale_log2;
          const bool rise = top > m + PX_SLACK || (x < 2 && top > m);
          if (__any_sync(FULL, rise)) {
            const float nm = rise ? top : m;
            const float k = rise ? ex2(m - nm) : 1.0f;  // 0 from -inf
            l *= k;
            lr *= k;
            m = nm;
            if (x >= 2) {
              // the product before is this warpgroup's unit before: two buffers back
              ok = __all_sync(FULL, wait(&o_done[buffer >= 2 ? buffer - 2 : buffer - 2 + BUFFERS], buffer >= 2 ? parity : parity ^ 1u));
              if (!ok) break;
              tc_fence_after();
#pragma unroll 1
              for (int y = 0; y < D / 16; ++y) {
                uint32_t v[16];
                tmem_ld16(to + static_cast<uint32_t>(16 * y), v);
#pragma unroll
                for (int z = 0; z < 16; ++z) v[z] = __float_as_uint(__uint_as_float(v[z]) * k);
                tmem_st16(to + static_cast<uint32_t>(16 * y), v);
              }
              tmem_st_wait();
            }
          }
          uint32_t pk[KEYS / 2];
          const float base = m == -INFINITY ? 0.0f : m;
          const float2 sc = make_float2(a.scale_log2, a.scale_log2), nb = make_float2(-base, -base);
          float2 sum0 = make_float2(0.0f, 0.0f), sum1 = sum0, rounded0 = sum0, rounded1 = sum0;
#pragma unroll
          for (int z = 0; z < KEYS / 2; ++z) {
            float2 p = __ffma2_rn(make_float2(f(2 * z), f(2 * z + 1)), sc, nb);
            p.x = ex2(p.x);
            p.y = ex2(p.y);
            if (z & 1) sum1 = __fadd2_rn(sum1, p); else sum0 = __fadd2_rn(sum0, p);
            pk[z] = pack2<BF16>(p.x, p.y);
            if (z & 1) add_rounded<BF16>(rounded1, pk[z]); else add_rounded<BF16>(rounded0, pk[z]);
          }
          tmem_st32(place, pk);
          if (pending) {  // the sums given at the end of the last shared tile
            ok = __all_sync(FULL, wait(taken, static_cast<uint32_t>(shared - 1) & 1u));
            if (!ok) break;
            pending = false;
          }
          tc_fence_before();
          mbar_arrive(&p_full[buffer]);
          l += (sum0.x + sum1.x) + (sum0.y + sum1.y);
          lr += (rounded0.x + rounded1.x) + (rounded0.y + rounded1.y);
          last_buffer = buffer, last_parity = parity;
          buffer += 2;
          if (buffer >= BUFFERS) buffer -= BUFFERS, parity ^= 1u;
        }
        if (!ok) break;
        ok = __all_sync(FULL, wait(&o_done[last_buffer], last_parity));
        if (!ok) break;
        tc_fence_after();
        if (own == CH_UNSEEN) m = -INFINITY, l = lr = 0.0f;
        float even = lr > 0.0f ? l / lr : 1.0f;  // O times this: what the unrounded p would have summed, but for its direction
        float other = 0.0f;                      // the same for the other warpgroup's O
        const bool both = !alone && end > 1;
        if (both) {
          ++shared;
          if (turn) {  // it has this one's sums: m, l and the sum of the rounded p here, O where it is
            s_ml[3 * row] = m, s_ml[3 * row + 1] = l, s_ml[3 * row + 2] = lr;
            mbar_arrive(given);
            pending = true;
            continue;
          }
          ok = __all_sync(FULL, wait(given, static_cast<uint32_t>(shared - 1) & 1u));
          if (!ok) break;
          tc_fence_after();
          const float m2 = s_ml[3 * row], l2 = s_ml[3 * row + 1], lr2 = s_ml[3 * row + 2];
          const float nm = fmaxf(m, m2), base = nm == -INFINITY ? 0.0f : nm, k = ex2(m - base), k2 = ex2(m2 - base);
          even = l == 0.0f ? 0.0f : even * k;
          other = l2 == 0.0f ? 0.0f : (lr2 > 0.0f ? l2 / lr2 : 1.0f) * k2;
          m = nm;
          l = l * k + l2 * k2;
        }
        // out = O / (sum of the rounded p); a part: O times l over that sum, with m and l
        const bool whole = g.slot < 0;
        if (whole) {
          const float inv = chunk_inverse(l);
          even *= inv;
          other *= inv;
        }
        const int token = tile * c.per_tile + row / a.G, gq = row % a.G;
        const bool exists = row < c.per_tile * a.G && token < g.tokens, sees = own != CH_UNSEEN;
        const int64_t out_at = static_cast<int64_t>(g.token + token) * a.ot + (static_cast<int64_t>(g.h) * a.G + gq) * a.oh;
        const int part_row = tile * c.per_tile * a.G + row;
        const uint32_t to2 = ts + static_cast<uint32_t>(BUFFERS * KEYS + D * (i ^ 1));
        float odd = 0.0f;  // a NaN where a value is not finite
#pragma unroll 1
        for (int y = 0; y < D / 32; ++y) {
          float v[32];
          tmem_ld32(to + static_cast<uint32_t>(32 * y), v);
#pragma unroll
          for (int x = 0; x < 32; ++x) {
            odd = fmaf(v[x], 0.0f, odd);  // (a NaN from an infinity, too)
            v[x] = l == 0.0f || even == 0.0f ? 0.0f : v[x] * even;  // (0 times what nobody saw)
          }
          if (both) {
            float z[32];
            tmem_ld32(to2 + static_cast<uint32_t>(32 * y), z);
#pragma unroll
            for (int x = 0; x < 32; ++x) {
              odd = fmaf(z[x], 0.0f, odd);
              v[x] = other == 0.0f ? v[x] : fmaf(z[x], other, v[x]);
            }
          }
          if (exists) {
            if (whole) {
              uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + out_at + 32 * y);
#pragma unroll
              for (int x = 0; x < 4; ++x)
                dst[x] = make_uint4(pack2<BF16>(v[8 * x], v[8 * x + 1]), pack2<BF16>(v[8 * x + 2], v[8 * x + 3]),
                                    pack2<BF16>(v[8 * x + 4], v[8 * x + 5]), pack2<BF16>(v[8 * x + 6], v[8 * x + 7]));
            } else {
              float4* dst = reinterpret_cast<float4*>(c.part_o) + (static_cast<int64_t>(g.slot) * (D / 4) + 8 * y) * c.slot_rows + part_row;
#pragma unroll
              for (int x = 0; x < 8; ++x) dst[x * c.slot_rows] = make_float4(v[4 * x], v[4 * x + 1], v[4 * x + 2], v[4 * x + 3]);
            }
          }
        }
        tc_fence_before();  // O has been read: the next P (its barrier) lets the next product into it start
        if (both) mbar_arrive(taken);
        if (exists) {
          if (!whole) c.part_ml[static_cast<int64_t>(g.slot) * c.slot_rows + part_row] = make_float2(m, l);
          else if (a.lse) a.lse[static_cast<int64_t>(g.token + token) * a.Hq + g.h * a.G + gq] = chunk_lse(m, l);
        }
        // sums that are not finite though the scores are: V holds an infinity or a NaN
        unsigned redo = __ballot_sync(FULL, sees && odd != odd && l > 0.0f && l < INFINITY);
        while (redo) {
          const int src = __ffs(redo) - 1;
          redo &= redo - 1;
          const int tk = __shfl_sync(FULL, token, src), q = __shfl_sync(FULL, gq, src), ow = __shfl_sync(FULL, own, src);
          const int fi = __shfl_sync(FULL, from, src);
          const int64_t oat = __shfl_sync(FULL, out_at, src);
          const int pr = __shfl_sync(FULL, part_row, src);
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
            for (int x = 0; x < E; ++x) {
              const int d = lane * E + x;
              c.part_o[((static_cast<int64_t>(g.slot) * (D / 4) + d / 4) * c.slot_rows + pr) * 4 + d % 4] = acc[x];
            }
            if (lane == 0) c.part_ml[static_cast<int64_t>(g.slot) * c.slot_rows + pr] = make_float2(km, kl);
          }
        }
      }
      __syncthreads();  // the segments have been taken, the next ones may be listed
      if (*reinterpret_cast<volatile int*>(failed)) break;
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(CH_REGS_OTHER));
    if (w == 0) {
      int copies = 0, v_copies = 0, q_copies = 0, bad = 0;  // (V's may be one behind K's where a wait gave up)
      for (bool again = works; again;) {
        chunk_walk(c, cta, s_rows, walker, s_segs, s_list, lanes_of_warp);
        __syncthreads();  // the segments are listed
        const int n = *s_segs;
        again = walker->more != 0;
        // ---- copies: lane l copies box l of a step (a page, or 128 tokens of one) ----
        const int rows = min(a.bs, CH_KEYS), pages = CH_KEYS / rows;
        auto key_of = [&](const ChunkSeg& g, int j) {  // the box's first key, of the prefix or of the row's own; -1: there is none
          const int s = g.step0 + j;
          const bool prefix = s < before;
          const int key = (prefix ? s : s - before) * CH_KEYS + lane * rows;
          return lane < pages && key < (prefix ? a.L : g.len) ? key : -1;
        };
        auto block_of = [&](const ChunkSeg& g, int j) {  // past the cache (it reads as zeros) where there is none
          const int key = key_of(g, j);
          if (key < 0) return a.blocks;
          const int32_t* ids = g.step0 + j < before ? a.prefix_blocks : a.table + g.b * a.table_stride;
          return ids[key >> a.bs_log2];
        };
        auto copy = [&](const CUtensorMap* map, unsigned char* ring, uint64_t* full, int s, int h, int block) {
          const int place = (lane * rows) & (a.bs - 1);
          if (lane == 0) mbar_expect_tx(&full[s], Tile::KV_BYTES);
          __syncwarp();
          if (lane < pages)
            for (int x = 0; x < HALVES; ++x)
              tma_load_slice(smem_u32(ring + s * Tile::KV_BYTES + x * CH_KEYS * 128 + lane * rows * 128), map, x, place, h, block, &full[s]);
        };
        int next = n ? block_of(s_list[0], 0) : 0;
        for (int e = 0; ok && e < n; ++e) {
          const ChunkSeg& g = s_list[e];
          const int steps = g.steps, h = g.h, tiles = tiles_of(g);
          for (int j = 0; ok && j < steps; ++j) {
            const bool inside = static_cast<unsigned>(next) < static_cast<unsigned>(a.blocks);
            bad |= !inside && key_of(g, j) >= 0;
            const int block = inside ? next : a.blocks;
            if (j + 1 < steps) next = block_of(g, j + 1);
            else if (e + 1 < n) next = block_of(s_list[e + 1], 0);
            const int s = copies % STAGES;
            const uint32_t parity = static_cast<uint32_t>(copies / STAGES - 1) & 1u;
            if (copies >= STAGES && !(ok = __all_sync(FULL, wait(&k_empty[s], parity)))) break;
            copy(&tm_k, s_k, k_full, s, h, block);
            ++copies;
            if (j == 0) {
              for (int i = 0; i < tiles; ++i) {
                const int place = q_copies & 1;
                if (q_copies >= 2 && !(ok = __all_sync(FULL, wait(&q_empty[place], static_cast<uint32_t>((q_copies >> 1) - 1) & 1u)))) break;
                if (lane == 0) {
                  mbar_expect_tx(&q_full[place], static_cast<uint32_t>(HALVES * c.per_tile * a.G * 128));
                  for (int x = 0; x < HALVES; ++x)
                    tma_load_3d(smem_u32(s_q + place * Tile::Q_BYTES + x * CH_M * 128), &tm_q, 64 * x, h * a.G, g.token + i * c.per_tile,
                                &q_full[place]);
                }
                __syncwarp();
                ++q_copies;
              }
              if (!ok) break;
            }
            if (copies > STAGES && !(ok = __all_sync(FULL, wait(&v_empty[s], parity)))) break;
            copy(&tm_v, s_v, v_full, s, h, block);
            ++v_copies;
          }
        }
        __syncthreads();  // the segments have been taken, the next ones may be listed
        if (*reinterpret_cast<volatile int*>(failed)) break;
      }
      if (bad && a.error_word) atomicOr(a.error_word, Q3S_DECERR_BLOCK_ID);
      // no copy may be in flight when the CTA leaves: wait for each place's last one
      if (lane == 0) {
        for (int i = max(0, q_copies - 2); i < q_copies; ++i) (void)mbar_wait_bounded(&q_full[i & 1], static_cast<uint32_t>(i >> 1) & 1u);
        for (int i = max(0, copies - STAGES); i < copies; ++i)
          (void)mbar_wait_bounded(&k_full[i % STAGES], static_cast<uint32_t>(i / STAGES) & 1u);
        for (int i = max(0, v_copies - STAGES); i < v_copies; ++i)
          (void)mbar_wait_bounded(&v_full[i % STAGES], static_cast<uint32_t>(i / STAGES) & 1u);
      }
    } else {
      // ---- products: warp 1 the second one, O += P V, warps 2 and 3 the scores of a softmax warpgroup each ----
      // (one warp for all scores took 450 clocks to issue a unit's eight products beside the softmax warps and 500 more for
      // its waits and loop: 2 rows of 4096 tokens 271 us, with two 244)
      constexpr uint32_t FMT = BF16 ? 1u : 0u;
      constexpr uint32_t ID_S = (1u << 4) | (FMT << 7) | (FMT << 10) | (static_cast<uint32_t>(KEYS >> 3) << 17) |
                                (static_cast<uint32_t>(CH_M >> 4) << 24);
      constexpr uint32_t ID_O = (1u << 4) | (FMT << 7) | (FMT << 10) | (1u << 16) | (static_cast<uint32_t>(D >> 3) << 17) |
                                (static_cast<uint32_t>(CH_M >> 4) << 24);  // bit 16: B's rows are the contraction
      constexpr uint64_t DESC_HI = (1024ull >> 4 << 32) | (1ull << 46) | (2ull << 61);  // of both kinds of descriptor
      const uint32_t leader = elect_one() ? 1u : 0u;
      const uint32_t q_lo = static_cast<uint32_t>(head_smem_desc(smem_u32(s_q))), k_lo = static_cast<uint32_t>(head_smem_desc(smem_u32(s_k)));
      const uint32_t v_lo = static_cast<uint32_t>(v_smem_desc(smem_u32(s_v)));
      for (bool again = works; again;) {
        __syncthreads();  // the segments are listed
        const int n = *s_segs;
        again = walker->more != 0;
        for (int e = 0; ok && e < n; ++e) {
          const int steps = s_list[e].steps, tiles = tiles_of(s_list[e]);
          const bool alone = tiles == 2;
          const int end = steps * PIECES * tiles, stride = w == 1 ? 1 : 2;
          const int x0 = w == 1 ? 0 : (w - units) & 1;  // warp 2 has the even units
          int buffer = (units + x0) % BUFFERS;
          uint32_t parity = static_cast<uint32_t>((units + x0) / BUFFERS) & 1u;
          bool used = units + x0 >= BUFFERS;  // the buffer, before
          int stage = kv % STAGES, step = -1;
          uint32_t stage_parity = static_cast<uint32_t>(kv / STAGES) & 1u;
          for (int x = x0; x < end; x += stride) {
            const int piece = alone ? x >> 1 : x, part = piece % PIECES;
            if (piece / PIECES != step) {
              if (step >= 0 && ++stage == STAGES) stage = 0, stage_parity ^= 1u;
              step = piece / PIECES;
              ok = __all_sync(FULL, wait(w == 1 ? &v_full[stage] : &k_full[stage], stage_parity));
              if (!ok) break;
            }
            if (w == 1) {
              ok = __all_sync(FULL, wait(&p_full[buffer], parity));
              if (!ok) break;
              tc_fence_after();
              const uint32_t dv = v_lo + static_cast<uint32_t>(stage * (Tile::KV_BYTES >> 4) + part * ((KEYS * 128) >> 4));
              const uint32_t to = tmem + static_cast<uint32_t>(BUFFERS * KEYS + D * ((units + x) & 1)), p = tmem + static_cast<uint32_t>(KEYS * buffer);
              const bool first = x < 2;  // into this O
#pragma unroll
              for (int k = 0; k < KEYS / 16; ++k)
                umma_ts_if(leader, to, p + static_cast<uint32_t>(8 * k), DESC_HI | (dv + static_cast<uint32_t>(k * ((16 * 128) >> 4))), ID_O, !first || k != 0);
              umma_commit_if(leader, &o_done[buffer]);
              if (part == PIECES - 1 && (!alone || (x & 1))) umma_commit_if(leader, &v_empty[stage]);
              if (++buffer == BUFFERS) buffer = 0, parity ^= 1u;
            } else {
              const uint32_t tile_q = static_cast<uint32_t>(tiles_q + (alone ? x & 1 : 0)), q = tile_q & 1u;
              if (x < 2) ok = __all_sync(FULL, wait(&q_full[q], (tile_q >> 1) & 1u));
              // the probabilities that were there have been taken
              if (ok && used) ok = __all_sync(FULL, wait(&o_done[buffer], parity ^ 1u));
              if (!ok) break;
              tc_fence_after();
              const uint32_t to = tmem + static_cast<uint32_t>(KEYS * buffer), dq = q_lo + q * static_cast<uint32_t>(Tile::Q_BYTES >> 4);
              const uint32_t dk = k_lo + static_cast<uint32_t>(stage * (Tile::KV_BYTES >> 4) + part * ((KEYS * 128) >> 4));
#pragma unroll
              for (int k = 0; k < D / 16; ++k) {
                constexpr int SLICE = (CH_KEYS * 128) >> 4;
                umma_ss_if(leader, to, DESC_HI | (dq + static_cast<uint32_t>((k / 4) * SLICE + (k % 4) * 2)),
                           DESC_HI | (dk + static_cast<uint32_t>((k / 4) * SLICE + (k % 4) * 2)), ID_S, k != 0);
              }
              umma_commit_if(leader, &s_full[buffer]);
              // each of the two warps frees a stage, and a tile of Q (one that only this warp has twice)
              if (!alone || part == PIECES - 1) umma_commit_if(leader, &k_empty[stage]);
              if (x + 2 >= end) {
                umma_commit_if(leader, &q_empty[q]);
                if (alone) umma_commit_if(leader, &q_empty[q]);
              }
              buffer += 2;
              if (buffer >= BUFFERS) buffer -= BUFFERS, parity ^= 1u, used = true;
            }
          }
          units += end;
          kv += steps;
          tiles_q += tiles;
        }
        __syncthreads();  // the segments have been taken, the next ones may be listed
        if (*reinterpret_cast<volatile int*>(failed)) break;
      }
      if (*failed) umma_commit_if(leader, done);  // products may still be running
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (w == 1) {
    tc_fence_after();
    if (*failed) (void)mbar_wait_bounded(done, 0);  // (bounded) before the columns go
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
  if (t == 0 && *failed && a.error_word) atomicOr(a.error_word, Q3S_DECERR_WAIT);
}

// A query row of a cut item (8 rows a warp) and TILES times 4 dims of it a lane, 16 dims apart, the first at `dim`:
// PARTS of its parts requested at a time.
template <int D, bool BF16, int TILES, int PARTS>
Q3S_DEV void chunk_join_row(const ChunkArgs& c, const ChunkCut& k, int r, int dim) {
  const AttnArgs& a = c.a;
  float4 acc[TILES];
  float m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < TILES; ++i) acc[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int p = 0; p < k.parts; p += PARTS) {
    float4 y[PARTS][TILES];
    float2 ml[PARTS];
#pragma unroll
    for (int j = 0; j < PARTS; ++j) {
      const int64_t slot = p + j == 0 ? k.slot : 2 * (k.cta + p + j);
      const bool live = p + j < k.parts;
      ml[j] = live ? c.part_ml[slot * c.slot_rows + r] : make_float2(-INFINITY, 0.0f);
#pragma unroll
      for (int i = 0; i < TILES; ++i)
        y[j][i] = live ? reinterpret_cast<const float4*>(c.part_o)[(slot * (D / 4) + dim / 4 + 4 * i) * c.slot_rows + r]
                       : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
#pragma unroll
    for (int j = 0; j < PARTS; ++j) {
      const float nm = fmaxf(m, ml[j].x), base = nm == -INFINITY ? 0.0f : nm;
      const float wm = ex2(m - base), wp = ex2(ml[j].x - base);
      m = nm;
      l = l * wm + wp * ml[j].y;
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
        acc[i].x = acc[i].x * wm + wp * y[j][i].x;
        acc[i].y = acc[i].y * wm + wp * y[j][i].y;
        acc[i].z = acc[i].z * wm + wp * y[j][i].z;
        acc[i].w = acc[i].w * wm + wp * y[j][i].w;
      }
    }
  }
  const int64_t token = k.token + r / a.G;
  const int head = k.h * a.G + r % a.G;
  const float inv = chunk_inverse(l);
#pragma unroll
  for (int i = 0; i < TILES; ++i)
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + token * a.ot + head * a.oh + dim + 16 * i) =
        make_uint2(pack2<BF16>(acc[i].x * inv, acc[i].y * inv), pack2<BF16>(acc[i].z * inv, acc[i].w * inv));
  if (a.lse && dim == 0) a.lse[token * a.Hq + head] = chunk_lse(m, l);
}

// Joins the parts of the items that were cut: 32 query rows a CTA, a warp 8 of them and half the dims, four parts at
// once (most items have two; eight parts, 16 dims at a time: 1 row of 300 tokens, 20000 keys, 87 us against 81).  Blocks behind those
// write 0 and -inf for the tokens that no item has (of no row, or that see nothing).  Bound by latency.
template <int D, bool BF16>
__global__ void __launch_bounds__(CH_JOIN_NT) attn_chunk_join_kernel(const ChunkArgs c, int join_blocks, int blocks_each) {
  const AttnArgs& a = c.a;
  const int t = static_cast<int>(threadIdx.x), w = t >> 5, lane = t & 31, block = static_cast<int>(blockIdx.x);
  constexpr int WARPS = CH_JOIN_NT / 32;
  grid_wait();
  grid_release();
  if (block < join_blocks) {
    const ChunkCut k = c.cuts[block / blocks_each];
    if (k.parts == 0) return;
    const int row0 = (block % blocks_each) * CH_JOIN_ROWS, rows = min(k.tokens * a.G, row0 + CH_JOIN_ROWS);
    static_assert(CH_JOIN_ROWS == 8 * WARPS / 2, "a warp's rows");
    const int r = row0 + (w & 3) * 8 + (lane & 7), dim = (w >> 2) * (D / 2) + (lane >> 3) * 4;
    if (r >= rows) return;
    constexpr int TILES = D / 32;
    chunk_join_row<D, BF16, TILES, 4>(c, k, r, dim);
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
