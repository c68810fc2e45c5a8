// q3s_attn_prefix.cuh -- the shared prefix for many queries, on the tensor
// cores (tcgen05): every query of the batch against the same keys.
#pragma once

#include <cuda.h>

#include "q3s_attn.cuh"
#include "q3s_head.cuh"

namespace q3s {

constexpr int PX_M = 128;       // query rows of a tile: the matrix instruction's M
constexpr int PX_KEYS = 128;    // keys of a step
constexpr int PX_STAGES = 2;    // steps of K (and of V) in shared memory
constexpr int PX_NT = 320;      // two softmax warpgroups (a tile each), the copy warp, the matrix warp
constexpr float PX_SLACK = 8.0f;  // log2 units that the running maximum may lag behind

template <int D>
struct PrefixTile {
  static constexpr int HALVES = D / 64;                   // 64-element (128-byte) slices of a row
  static constexpr int Q_BYTES = PX_M * D * 2;
  static constexpr int KV_BYTES = PX_KEYS * D * 2;
  static constexpr int USED = 1024 + 2 * Q_BYTES + 2 * PX_STAGES * KV_BYTES + 256;
  static constexpr int SMEM = USED > TMEM_ALL_SMEM ? USED : TMEM_ALL_SMEM;  // all of the tensor memory
};

struct PrefixArgs {
  AttnArgs a;
  int per_tile;   // tokens of a tile: 128 / G
  int steps;      // ceil(L / 128)
  int per_split;  // steps of a part
};

Q3S_DEV void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
// Part of one block of a cache, 64 dims (slice x).
Q3S_DEV void tma_load_slice(uint32_t dst, const CUtensorMap* map, int x, int place, int h, int block, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::
          "r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(place), "r"(x), "r"(h), "r"(block), "r"(smem_u32(bar))
      : "memory");
}
// D += A B with A from TMEM.
Q3S_DEV void umma_f16_ta(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate));
}
// Shared-memory descriptor of V as the product's B operand: rows are keys (the
// contraction), 128 bytes of 64 dims each, 128-byte swizzle.  The next 64 dims
// are one slice (128 keys * 128 bytes) away (leading byte offset), the next 8
// keys 1024 bytes (stride byte offset).
Q3S_DEV uint64_t v_smem_desc(uint32_t saddr) {
  return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>((PX_KEYS * 128) >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// One lane of a converged warp (the compiler then knows that the branch is taken by one thread).
Q3S_DEV bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n}" : "=r"(p));
  return p != 0;
}
// 128 consecutive 32-bit columns of this thread's TMEM lane.
Q3S_DEV void tmem_ld128(uint32_t addr, uint32_t (&r)[128]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,"
      "%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63},"
      " [%128];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%64,%65,%66,%67,%68,%69,%70,%71,%72,%73,%74,%75,%76,%77,%78,"
      "%79,%80,%81,%82,%83,%84,%85,%86,%87,%88,%89,%90,%91,%92,%93,%94,%95,%96,%97,%98,%99,%100,%101,%102,"
      "%103,%104,%105,%106,%107,%108,%109,%110,%111,%112,%113,%114,%115,%116,%117,%118,%119,%120,%121,%122,"
      "%123,%124,%125,%126,%127}, [%128+64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
        "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
        "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63]),
        "=r"(r[64]), "=r"(r[65]), "=r"(r[66]), "=r"(r[67]), "=r"(r[68]), "=r"(r[69]), "=r"(r[70]), "=r"(r[71]),
        "=r"(r[72]), "=r"(r[73]), "=r"(r[74]), "=r"(r[75]), "=r"(r[76]), "=r"(r[77]), "=r"(r[78]), "=r"(r[79]),
        "=r"(r[80]), "=r"(r[81]), "=r"(r[82]), "=r"(r[83]), "=r"(r[84]), "=r"(r[85]), "=r"(r[86]), "=r"(r[87]),
        "=r"(r[88]), "=r"(r[89]), "=r"(r[90]), "=r"(r[91]), "=r"(r[92]), "=r"(r[93]), "=r"(r[94]), "=r"(r[95]),
        "=r"(r[96]), "=r"(r[97]), "=r"(r[98]), "=r"(r[99]), "=r"(r[100]), "=r"(r[101]), "=r"(r[102]),
        "=r"(r[103]), "=r"(r[104]), "=r"(r[105]), "=r"(r[106]), "=r"(r[107]), "=r"(r[108]), "=r"(r[109]),
        "=r"(r[110]), "=r"(r[111]), "=r"(r[112]), "=r"(r[113]), "=r"(r[114]), "=r"(r[115]), "=r"(r[116]),
        "=r"(r[117]), "=r"(r[118]), "=r"(r[119]), "=r"(r[120]), "=r"(r[121]), "=r"(r[122]), "=r"(r[123]),
        "=r"(r[124]), "=r"(r[125]), "=r"(r[126]), "=r"(r[127])
      : "r"(addr)
      : "memory");
}

// 64 consecutive columns.
Q3S_DEV void tmem_ld64(uint32_t addr, uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,"
      "%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
        "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
        "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(addr)
      : "memory");
}

// 64 columns written; the store is complete when it returns.
Q3S_DEV void tmem_st64(uint32_t addr, const uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x64.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,"
      "%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63,"
      "%64};\n\t"
      "tcgen05.wait::st.sync.aligned;" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(r[32]),
      "r"(r[33]), "r"(r[34]), "r"(r[35]), "r"(r[36]), "r"(r[37]), "r"(r[38]), "r"(r[39]), "r"(r[40]),
      "r"(r[41]), "r"(r[42]), "r"(r[43]), "r"(r[44]), "r"(r[45]), "r"(r[46]), "r"(r[47]), "r"(r[48]),
      "r"(r[49]), "r"(r[50]), "r"(r[51]), "r"(r[52]), "r"(r[53]), "r"(r[54]), "r"(r[55]), "r"(r[56]),
      "r"(r[57]), "r"(r[58]), "r"(r[59]), "r"(r[60]), "r"(r[61]), "r"(r[62]), "r"(r[63])
      : "memory");
}

// 32 columns written; the store is complete when it returns.
Q3S_DEV void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};\n\t"
      "tcgen05.wait::st.sync.aligned;" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

// Largest of three.
Q3S_DEV float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// One CTA: 2 * 128 query rows of one key/value head over one part of the
// prefix.  Rows of a tile are (token, head of the group) pairs, so a group's
// heads share the keys that are read.
//
// The matrix warp alternates between the two tiles,
//   S0 = Q0 K^T, S1 = Q1 K^T, then per step  O0 += P0 V, S0 = Q0 K'^T, O1 += P1 V, S1 = Q1 K'^T,
// so that one tile's softmax runs while the other tile's products do.  A
// softmax thread owns a row: it reads the 128 scores from TMEM, writes p over
// them as 16-bit values (the second product's A operand, straight from TMEM) in
// two halves, so that the product starts on the first while the second is
// computed, and keeps m and l in registers.  TMEM: S0 S1 O0 O1, 128 columns each.
//
// The running maximum is allowed to lag by 8 (p up to 256, sums in fp32), so
// O is rescaled only when a score rises above that: the first step sets it,
// later ones almost never.  The product takes p rounded to 16 bits.  l sums the
// unrounded p, for the log-sum-exp and the join, and a second sum the rounded
// ones: O is divided by that one (times l) at the end, so that a rounding moves
// the result by p |v - out|, not p |v|: next to nothing where one key carries the
// row, and over many keys it averages out (the other kernel, for few keys, holds
// p in two parts).  With U the type's unit roundoff the result is off by
// U |out| + U sum p |v - out|.  The second sum costs three instructions a pair of
// keys (the 256 rows below 92 us in place of 88; in one chain 93).
//
// Keys past the end: whole boxes read as zeros (an out-of-range block
// coordinate), the rest of the last one is cleared in V and masked in S.
// Bound by the exponentials (16 a clock and SM: 1024 clocks for 128 x 128
// scores) and, equally, by the two products (1024 clocks at the tensor peak):
// 256 rows of 4 x 8 heads on 16000 keys of 128 (67 GFLOP, 41 us at the peak of a
// large product) take 79 us, 54% of the tensor pipe (the whole operator 92 us in a burst and
// 107 in seconds of it, at the power limit and 1.66 GHz).  Some of the exponentials as
// polynomials made it slower (90 to 95 us with the rest of the operator, 88.7
// without): the two products in the shape 128 x 128 x 16 are near what they
// reach.  One tile a CTA where that fills more SMs was no faster either: from 2.5
// us less to 8 more, as the key-split kernel beside it loses those SMs.
template <int D, bool BF16>
__global__ void __launch_bounds__(PX_NT, 1)
    attn_prefix_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, const PrefixArgs p) {
  using Tile = PrefixTile<D>;
  constexpr int HALVES = Tile::HALVES;
  const AttnArgs& a = p.a;
  extern __shared__ __align__(1024) unsigned char px_smem[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(px_smem) + 1023) &
                                                         ~static_cast<uintptr_t>(1023));
  unsigned char* s_q = smem;
  unsigned char* s_k = s_q + 2 * Tile::Q_BYTES;
  unsigned char* s_v = s_k + PX_STAGES * Tile::KV_BYTES;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(s_v + PX_STAGES * Tile::KV_BYTES);
  uint64_t* k_full = q_full + 1;
  uint64_t* k_empty = k_full + PX_STAGES;
  uint64_t* v_full = k_empty + PX_STAGES;
  uint64_t* v_empty = v_full + PX_STAGES;
  uint64_t* s_full = v_empty + PX_STAGES;  // [2] scores of a tile are in TMEM
  uint64_t* p_half = s_full + 2;           // [2] the probabilities of its first 64 keys are
  uint64_t* p_full = p_half + 2;           // [2] all are
  uint64_t* o_done = p_full + 2;           // [2] its second product is complete
  uint64_t* v_clean = o_done + 2;          // V of a part's ragged last step has been cleared past its end
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(v_clean + 1);
  int* failed = reinterpret_cast<int*>(tmem_slot + 1);
  const int t = static_cast<int>(threadIdx.x), w = t >> 5, lane = t & 31;
  const int pair = static_cast<int>(blockIdx.x), h = static_cast<int>(blockIdx.y), split = static_cast<int>(blockIdx.z);
  const int step0 = split * p.per_split, steps = min(p.per_split, p.steps - step0);  // >= 1
  const int token0 = pair * 2 * p.per_tile;
  const int tiles = token0 + p.per_tile < a.T ? 2 : 1;  // a last pair may have one tile

  // ---- copies: lane l copies box l of a step (a page, or 128 tokens of one) ----
  const int rows = min(a.bs, PX_KEYS), pages = PX_KEYS / rows;
  auto block_of = [&](int j) {  // lane's block of step j; past the cache (it reads as zeros) where there is none
    const int key = (step0 + j) * PX_KEYS + lane * rows;
    return j < steps && lane < pages && key < a.L ? a.prefix_blocks[key >> a.bs_log2] : a.blocks;
  };
  int bad = 0;
  auto copy = [&](const CUtensorMap* map, unsigned char* ring, uint64_t* full, int j, int block) {
    const bool inside = static_cast<unsigned>(block) < static_cast<unsigned>(a.blocks);
    bad |= !inside && block != a.blocks;
    const int id = inside ? block : a.blocks, place = ((step0 + j) * PX_KEYS + lane * rows) & (a.bs - 1), s = j % PX_STAGES;
    if (lane == 0) mbar_expect_tx(&full[s], Tile::KV_BYTES);
    __syncwarp();
    if (lane < pages)
      for (int x = 0; x < HALVES; ++x)
        tma_load_slice(smem_u32(ring + s * Tile::KV_BYTES + x * PX_KEYS * 128 + lane * rows * 128), map, x, place, h, id, &full[s]);
  };
  grid_wait();
  grid_release();  // the key-split kernel
  if (w == 8) {  // the first copies are on their way while TMEM is allocated
    if (lane < 3) prefetch_map(lane == 0 ? &tm_q : lane == 1 ? &tm_k : &tm_v);
    int block[PX_STAGES];
#pragma unroll
    for (int j = 0; j < PX_STAGES; ++j) block[j] = block_of(j);
    if (lane == 0) {
      mbar_init(q_full, 1);
      mbar_init(v_clean, 1);
      for (int s = 0; s < PX_STAGES; ++s) {
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
      mbar_expect_tx(q_full, static_cast<uint32_t>(tiles * HALVES * p.per_tile * a.G * 128));
      for (int i = 0; i < tiles; ++i)
        for (int x = 0; x < HALVES; ++x)
          tma_load_3d(smem_u32(s_q + i * Tile::Q_BYTES + x * PX_M * 128), &tm_q, 64 * x, h * a.G, token0 + i * p.per_tile, q_full);
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < PX_STAGES; ++j)
      if (j < steps) {
        copy(&tm_k, s_k, k_full, j, block[j]);
        copy(&tm_v, s_v, v_full, j, block[j]);
      }
  }
  if (w == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // a wait that gives up marks the CTA; every role then stops at its next wait
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*reinterpret_cast<volatile int*>(failed)) return false;
    if (mbar_wait_bounded(bar, parity)) return true;
    atomicOr(failed, 1);
    return false;
  };

  if (w == 8) {
    int next = block_of(PX_STAGES), j = min(PX_STAGES, steps);
    for (; j < steps; ++j) {
      const int block = next;
      next = block_of(j + 1);
      const int s = j % PX_STAGES;
      if (!__all_sync(FULL, wait(&k_empty[s], ((j / PX_STAGES) - 1) & 1))) break;
      copy(&tm_k, s_k, k_full, j, block);
      if (!__all_sync(FULL, wait(&v_empty[s], ((j / PX_STAGES) - 1) & 1))) break;
      copy(&tm_v, s_v, v_full, j, block);
    }
    if (bad && a.error_word) atomicOr(a.error_word, Q3S_DECERR_BLOCK_ID);
    const int valid = a.L - (step0 + steps - 1) * PX_KEYS;  // keys of the last step
    if (j == steps && valid < PX_KEYS) {  // clear V past the end, up to the end of its box
      const int last = steps - 1, s = last % PX_STAGES, end = (valid + rows - 1) / rows * rows;
      if (__all_sync(FULL, wait(&v_full[s], (last / PX_STAGES) & 1))) {
        for (int c = lane; c < (end - valid) * 8; c += 32)
          for (int x = 0; x < HALVES; ++x)
            *reinterpret_cast<uint4*>(s_v + s * Tile::KV_BYTES + x * PX_KEYS * 128 + valid * 128 + c * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(v_clean);
      }
    }
    // no copy may be in flight when the CTA leaves: wait for each stage's last one
    if (lane == 0) {
      (void)mbar_wait_bounded(q_full, 0);
      for (int i = max(0, j - PX_STAGES); i < j; ++i) {
        (void)mbar_wait_bounded(&k_full[i % PX_STAGES], (i / PX_STAGES) & 1);
        (void)mbar_wait_bounded(&v_full[i % PX_STAGES], (i / PX_STAGES) & 1);
      }
    }
  } else if (w == 9) {
    // ---- products --------------------------------------------------------------
    constexpr uint32_t FMT = BF16 ? 1u : 0u;
    constexpr uint32_t ID_S = (1u << 4) | (FMT << 7) | (FMT << 10) | (static_cast<uint32_t>(PX_KEYS >> 3) << 17) |
                              (static_cast<uint32_t>(PX_M >> 4) << 24);
    constexpr uint32_t ID_O = (1u << 4) | (FMT << 7) | (FMT << 10) | (1u << 16) | (static_cast<uint32_t>(D >> 3) << 17) |
                              (static_cast<uint32_t>(PX_M >> 4) << 24);  // bit 16: B's rows are the contraction
    if (elect_one()) {
      const uint64_t q_desc = head_smem_desc(smem_u32(s_q)), k_desc = head_smem_desc(smem_u32(s_k)), v_desc = v_smem_desc(smem_u32(s_v));
      auto scores = [&](int i, int s) {  // S_i = Q_i K^T
        const uint64_t dq = q_desc + static_cast<uint64_t>(i * (Tile::Q_BYTES >> 4)), dk = k_desc + static_cast<uint64_t>(s * (Tile::KV_BYTES >> 4));
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          constexpr int SLICE = (PX_KEYS * 128) >> 4;
          umma_f16(tmem + static_cast<uint32_t>(128 * i), dq + (c / 4) * SLICE + (c % 4) * 2, dk + (c / 4) * SLICE + (c % 4) * 2, ID_S, c != 0);
        }
        umma_commit(&s_full[i]);
      };
      bool ok = wait(q_full, 0) && wait(&k_full[0], 0);
      tc_fence_after();
      if (ok) {
        for (int i = 0; i < tiles; ++i) scores(i, 0);
        umma_commit(&k_empty[0]);
      }
      for (int j = 0; ok && j < steps; ++j) {
        const int s = j % PX_STAGES, s1 = (j + 1) % PX_STAGES;
        ok = wait(&v_full[s], (j / PX_STAGES) & 1);
        if (ok && j + 1 == steps && a.L < (step0 + steps) * PX_KEYS) ok = wait(v_clean, 0);
        for (int i = 0; ok && i < tiles; ++i) {
          const uint64_t dv = v_desc + static_cast<uint64_t>(s * (Tile::KV_BYTES >> 4));
#pragma unroll
          for (int half = 0; half < 2; ++half) {  // O_i += P_i V
            ok = ok && wait(half ? &p_full[i] : &p_half[i], j & 1);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < PX_KEYS / 32; ++c) {
              const int k = half * (PX_KEYS / 32) + c;
              umma_f16_ta(tmem + static_cast<uint32_t>(256 + 128 * i), tmem + static_cast<uint32_t>(128 * i + 8 * k),
                          dv + k * ((16 * 128) >> 4), ID_O, (j | k) != 0);
            }
          }
          if (!ok) break;
          if (i == tiles - 1) umma_commit(&v_empty[s]);
          umma_commit(&o_done[i]);
          if (j + 1 < steps) {
            if (i == 0) {
              ok = wait(&k_full[s1], ((j + 1) / PX_STAGES) & 1);
              if (!ok) break;
              tc_fence_after();
            }
            scores(i, s1);
            if (i == tiles - 1) umma_commit(&k_empty[s1]);
          }
        }
      }
    }
    __syncwarp();
  } else {
    // ---- softmax ----------------------------------------------------------------
    const int i = w >> 2, row = (w & 3) * 32 + lane;
    if (i < tiles) {
      const uint32_t lanes = static_cast<uint32_t>((w & 3) * 32) << 16;
      const uint32_t ts = tmem + lanes + static_cast<uint32_t>(128 * i), to = tmem + lanes + static_cast<uint32_t>(256 + 128 * i);
      float m = -INFINITY, l = 0.0f, lr = 0.0f;  // lr: of the rounded p
      bool ok = true;
      for (int j = 0; j < steps; ++j) {
        ok = __all_sync(FULL, wait(&s_full[i], j & 1));
        if (!ok) break;
        tc_fence_after();
        uint32_t r[128];
        tmem_ld128(ts, r);
        const int valid = a.L - (step0 + j) * PX_KEYS;
        if (valid < PX_KEYS) {
#pragma unroll
          for (int c = 0; c < 128; ++c)
            if (c >= valid) r[c] = 0xff800000u;
        }
        auto f = [&](int c) { return __uint_as_float(r[c]); };
        float x[4] = {f(0), f(1), f(2), f(3)};
#pragma unroll
        for (int c = 4; c + 8 <= 128; c += 8) {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = max3(x[e], f(c + 2 * e), f(c + 2 * e + 1));
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = fmaxf(x[e], f(124 + e));
        const float top = max3(fmaxf(x[0], x[1]), x[2], x[3]) * a.scale_log2;
        const bool rise = top > m + PX_SLACK || (j == 0 && top > m);
        if (__any_sync(FULL, rise)) {
          const float nm = rise ? top : m;
          const float c = rise ? ex2(m - nm) : 1.0f;  // 0 from -inf
          l *= c;
          lr *= c;
          m = nm;
          if (j > 0) {
            ok = __all_sync(FULL, wait(&o_done[i], (j - 1) & 1));
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int k = 0; k < D / 32; ++k) {
              float v[32];
              tmem_ld32(to + static_cast<uint32_t>(32 * k), v);
              uint32_t u[32];
#pragma unroll
              for (int e = 0; e < 32; ++e) u[e] = __float_as_uint(v[e] * c);
              tmem_st32(to + static_cast<uint32_t>(32 * k), u);
            }
          }
        }
        const float base = m == -INFINITY ? 0.0f : m;
        const float2 sc = make_float2(a.scale_log2, a.scale_log2), nb = make_float2(-base, -base);
        float2 sum0 = make_float2(0.0f, 0.0f), sum1 = sum0, rounded0 = sum0, rounded1 = sum0;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t pk[32];
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            float2 e = __ffma2_rn(make_float2(f(64 * half + 2 * c), f(64 * half + 2 * c + 1)), sc, nb);
            e.x = ex2(e.x);
            e.y = ex2(e.y);
            if (c & 1) sum1 = __fadd2_rn(sum1, e); else sum0 = __fadd2_rn(sum0, e);
            pk[c] = pack2<BF16>(e.x, e.y);
            const float2 r2 = unpack2<BF16>(pk[c]);
            if (c & 1) rounded1 = __fadd2_rn(rounded1, r2); else rounded0 = __fadd2_rn(rounded0, r2);
          }
          tmem_st32(ts + static_cast<uint32_t>(32 * half), pk);
          tc_fence_before();
          mbar_arrive(half ? &p_full[i] : &p_half[i]);
        }
        l += (sum0.x + sum1.x) + (sum0.y + sum1.y);
        lr += (rounded0.x + rounded1.x) + (rounded0.y + rounded1.y);
      }
      if (ok) ok = __all_sync(FULL, wait(&o_done[i], (steps - 1) & 1));
      if (ok) {
        tc_fence_after();
        // O through shared memory: a thread writes its row there (16 bytes of
        // padding a row keep that free of bank conflicts) and copies it out in one
        // piece.  Tile 0's rows take the place of tile 1's queries and of K, whose
        // last readers came before this tile's last product; tile 1's what follows.
        constexpr int PITCH = D * 4 + 16;
        static_assert(2 * PX_M * PITCH + 1024 <= Tile::Q_BYTES + 2 * PX_STAGES * Tile::KV_BYTES, "room for both tiles");
        static_assert(PX_M * PITCH <= Tile::Q_BYTES + PX_STAGES * Tile::KV_BYTES, "tile 0 leaves V alone");
        unsigned char* stage = s_q + Tile::Q_BYTES + i * PX_M * PITCH + row * PITCH;
        const float even = lr > 0.0f ? l / lr : 1.0f;
#pragma unroll 1
        for (int k = 0; k < D / 32; ++k) {
          float v[32];
          tmem_ld32(to + static_cast<uint32_t>(32 * k), v);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            *reinterpret_cast<float4*>(stage + (8 * k + e) * 16) = make_float4(v[4 * e] * even, v[4 * e + 1] * even, v[4 * e + 2] * even, v[4 * e + 3] * even);
        }
        const int token = token0 + i * p.per_tile + row / a.G;
        if (row < p.per_tile * a.G && token < a.T) {  // there is such a query row
          const int64_t at = (static_cast<int64_t>(split) * a.T + token) * a.Hq + h * a.G + row % a.G;
          fence_proxy_async_smem();
          asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(a.pre_o + at * D), "r"(smem_u32(stage)),
                       "r"(D * 4)
                       : "memory");
          a.pre_ml[at] = make_float2(m, l);
        }
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (w == 9) {
    tc_fence_after();
    if (*failed) {  // products may still be running: their commits (bounded) before the columns go
      if (lane == 0)
        for (int i = 0; i < 2; ++i) (void)mbar_wait_bounded(&o_done[i], 0);
      __syncwarp();
    }
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
  if (t == 0 && *failed && a.error_word) atomicOr(a.error_word, Q3S_DECERR_WAIT);
}

}  // namespace q3s
