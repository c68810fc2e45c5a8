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

#include <cuda_runtime.h>
#include <stdint.h>

#include "q3s_args.cuh"
#include "q3s_decode.h"
#include "q3s_device.cuh"

namespace q3s {

constexpr int AT_KEYS = 32;    // keys of a unit (one pipeline stage of a warp)
constexpr int AT_ROWS = 16;    // query rows of an item: the matrix instruction's M
constexpr int AT_WARPS = 4;
constexpr int AT_STAGES = 3;
constexpr int AT_MIN_UNITS = 2;  // fewest units a warp takes before another one is used

struct AttnArgs {
  int B, T, Hq, H, G, bs, blocks, max_blocks;
  int L;            // prefix tokens
  int prefix_here;  // 1: the key-split kernel computes the prefix too (as a row of all T tokens)
  int splits;       // parts of the prefix kernel (prefix_here == 0)
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
  // workspace
  int32_t* plan;     // {units per warp, warps}, then per row (row 0: the prefix) {first unit lo, hi, first item}
  float* part_o;     // [slots][16][D]
  float2* part_ml;   // [slots][16] (m in log2 units, l)
  int64_t slots;     // capacity
  float* pre_o;      // [splits][T * Hq][D]
  float2* pre_ml;    // [splits][T * Hq]
};

// Row r of the work list: r = 0 is the prefix seen by all T tokens (empty
// unless it is computed here), r = b + 1 the own tokens of batch row b.
struct AttnRow {
  int t0, n, len, causal;  // first token, tokens, keys; 1: token i sees keys j <= len - n + i
  int units, tiles;        // units of its keys, 16-row tiles of its n * G query rows
};
Q3S_DEV AttnRow attn_row(const AttnArgs& a, int r) {
  AttnRow x;
  if (r == 0) {
    x.t0 = 0;
    x.n = a.prefix_here ? a.T : 0;
    x.len = a.L;
    x.causal = 0;
  } else {
    const int o0 = a.offsets[r - 1], o1 = a.offsets[r], len = a.lengths[r - 1];
    x.t0 = min(max(o0, 0), a.T);
    x.n = min(max(o1, x.t0), a.T) - x.t0;
    x.len = static_cast<int>(min(static_cast<int64_t>(max(len, 0)), static_cast<int64_t>(a.max_blocks) * a.bs));
    x.causal = 1;
  }
  x.units = x.n > 0 ? (x.len + AT_KEYS - 1) / AT_KEYS : 0;
  x.tiles = x.units ? (static_cast<int>((static_cast<int64_t>(x.n) * a.G + AT_ROWS - 1) / AT_ROWS)) : 0;
  return x;
}

template <bool BF16>
Q3S_DEV void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
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
    float2 r;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n}"
        : "=f"(r.x), "=f"(r.y) : "r"(p));
    return r;
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
// 16 bytes global -> shared, zeros where !full (the source is then not read).
Q3S_DEV void cp16(uint32_t dst, const void* src, bool full) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(full ? 16 : 0) : "memory");
}

// Where a warp is in the work list.
struct AttnPos {
  int r, h, tile, u;  // row, kv head, query tile, unit of the row's keys
  AttnRow x;
  int item;           // items before this one
};
Q3S_DEV void attn_next(const AttnArgs& a, AttnPos& p) {
  if (++p.u < p.x.units) return;
  p.u = 0;
  ++p.item;
  if (++p.tile < p.x.tiles) return;
  p.tile = 0;
  if (++p.h < a.H) return;
  p.h = 0;
  do {
    if (++p.r > a.B) return;  // past the end: never read
    p.x = attn_row(a, p.r);
  } while (p.x.units == 0);
}

// The key-split kernel.  The keys of every (row, kv head, 16-row query tile)
// item are cut into units of 32; all units of the batch form one list, cut
// into equal contiguous ranges, one a warp, so that rows of any lengths load
// the GPU evenly with no more than one part per item plus one per warp.  Each
// CTA derives the list from the device's lengths (one scan of the rows), so no
// host plan is needed and a captured graph follows the lengths.
//
// A warp works alone: a three-stage cp.async ring of its own (keys past the
// end arrive as zeros, so nothing that lies there, NaN included, reaches the
// products), S = Q K^T and O += P V by the warp-level matrix instruction
// m16n8k16 with the 16 query rows as M.  With one query a row this is bound by
// reading the cache (2 * G useful operations a byte): the matrix instruction
// is there to keep the arithmetic under the loads, and the tcgen05 form, whose
// M is 128, would be nearly empty.  Many queries on a long prefix are the other
// kernel's. 
template <int D, bool BF16>
__global__ void __launch_bounds__(AT_WARPS * 32) attn_split_kernel(const AttnArgs a) {
  constexpr int CH = D / 8;                     // 16-byte chunks of a key
  constexpr int TILE = AT_KEYS * D * 2;         // bytes of a unit's keys (or values)
  constexpr int PER = AT_KEYS * CH / 32;        // chunks a lane copies
  constexpr int KEYS_PER = 32 / CH;             // keys a warp copies at a time
  extern __shared__ __align__(128) unsigned char at_smem[];
  __shared__ long long s_units[AT_WARPS * 32 + 1];
  __shared__ int s_items[AT_WARPS * 32 + 1];
  const int t = static_cast<int>(threadIdx.x), w = t >> 5, lane = t & 31;
  asm volatile("griddepcontrol.launch_dependents;");

  // ---- the work list -------------------------------------------------------
  // thread t sums rows [t * per, (t + 1) * per)
  const int rows = a.B + 1, NT = AT_WARPS * 32;
  const int per = (rows + NT - 1) / NT;
  long long mu = 0;
  int mi = 0;
  for (int i = 0; i < per; ++i) {
    const int r = t * per + i;
    if (r >= rows) break;
    const AttnRow x = attn_row(a, r);
    mu += static_cast<long long>(x.units) * x.tiles * a.H;
    mi += x.tiles * a.H;
  }
  s_units[t + 1] = mu;
  s_items[t + 1] = mi;
  if (t == 0) s_units[0] = 0, s_items[0] = 0;
  __syncthreads();
  if (w == 0) {  // exclusive scan of NT values, NT / 32 a lane
    long long u[AT_WARPS], su = 0;
    int it[AT_WARPS], si = 0;
#pragma unroll
    for (int k = 0; k < AT_WARPS; ++k) {
      su += s_units[1 + lane * AT_WARPS + k];
      si += s_items[1 + lane * AT_WARPS + k];
      u[k] = su;
      it[k] = si;
    }
    long long pu = su;
    int pi = si;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long ou = __shfl_up_sync(FULL, pu, d);
      const int oi = __shfl_up_sync(FULL, pi, d);
      if (lane >= d) pu += ou, pi += oi;
    }
    pu -= su;
    pi -= si;
#pragma unroll
    for (int k = 0; k < AT_WARPS; ++k) {
      s_units[1 + lane * AT_WARPS + k] = pu + u[k];
      s_items[1 + lane * AT_WARPS + k] = pi + it[k];
    }
  }
  __syncthreads();
  const long long all = s_units[NT];
  const long long warps = static_cast<long long>(gridDim.x) * AT_WARPS;
  const long long quota = max((all + warps - 1) / warps, static_cast<long long>(AT_MIN_UNITS));
  if (blockIdx.x == 0) {  // the plan, for the kernel that joins the parts
    if (t == 0) reinterpret_cast<long long*>(a.plan)[0] = quota;
    long long u = s_units[t];
    int it = s_items[t];
    int bad = 0;
    for (int i = 0; i < per; ++i) {
      const int r = t * per + i;
      if (r >= rows) break;
      const AttnRow x = attn_row(a, r);
      reinterpret_cast<long long*>(a.plan)[1 + r] = u;
      a.plan[2 * (1 + rows) + r] = it;
      u += static_cast<long long>(x.units) * x.tiles * a.H;
      it += x.tiles * a.H;
      if (r > 0 && (a.lengths[r - 1] != x.len || a.offsets[r - 1] != x.t0 || a.offsets[r] != x.t0 + x.n))
        bad = Q3S_DECERR_LENGTHS;
    }
    if (bad && a.error_word) atomicOr(a.error_word, bad);
  }
  // this warp's range: warps of a CTA are neighbours in the list
  const long long gw = static_cast<long long>(blockIdx.x) * AT_WARPS + w;
  const long long u0 = gw * quota, u1 = min(u0 + quota, all);
  if (u0 >= u1) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }

  AttnPos p;
  {
    int l = 0, r = NT;  // the last thread chunk that starts at or before u0
    while (r - l > 1) {
      const int m = (l + r) >> 1;
      if (s_units[m] <= u0) l = m; else r = m;
    }
    long long at = s_units[l];
    p.item = s_items[l];
    p.r = l * per;
    for (;; ++p.r) {
      p.x = attn_row(a, p.r);
      const long long n = static_cast<long long>(p.x.units) * p.x.tiles * a.H;
      if (u0 < at + n) break;
      at += n;
      p.item += p.x.tiles * a.H;
    }
    const long long d = u0 - at;
    const int in = static_cast<int>(d / p.x.units);  // item within the row
    p.u = static_cast<int>(d - static_cast<long long>(in) * p.x.units);
    p.h = in / p.x.tiles;
    p.tile = in - p.h * p.x.tiles;
    p.item += in;
  }

  const uint32_t ring = smem_u32(at_smem) + static_cast<uint32_t>(w * AT_STAGES * 2 * TILE);
  const int total = static_cast<int>(u1 - u0);
  int bad_block = 0;

  // ---- producer: unit -> ring stage ----------------------------------------
  AttnPos pf = p;  // the next unit to fetch
  auto block_of = [&](const AttnPos& q) {  // lane l: the cache block of key l of the unit (-1: none)
    const int j = q.u * AT_KEYS + lane;
    if (j >= q.x.len) return -1;
    const int id = q.r == 0 ? a.prefix_blocks[j / a.bs] : a.table[(q.r - 1) * a.table_stride + j / a.bs];
    if (static_cast<unsigned>(id) < static_cast<unsigned>(a.blocks)) return id;
    bad_block = 1;
    return -1;
  };
  int next_id = block_of(pf);
  int fetched = 0;
  auto fetch = [&]() {
    if (fetched < total) {
      const uint32_t dst = ring + static_cast<uint32_t>((fetched % AT_STAGES) * 2 * TILE);
      const int place = (pf.u * AT_KEYS + lane) % a.bs;
      const bool have = next_id >= 0;
      const int64_t ko = have ? next_id * a.kb + pf.h * a.kh + place * a.kp : 0;
      const int64_t vo = have ? next_id * a.vb + pf.h * a.vh + place * a.vp : 0;
      const uint32_t got = __ballot_sync(FULL, have);
      const int c = lane % CH;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int key = i * KEYS_PER + lane / CH;
        const int64_t k0 = __shfl_sync(FULL, ko, key), v0 = __shfl_sync(FULL, vo, key);
        const bool full = (got >> key) & 1;
        const uint32_t at = static_cast<uint32_t>(key * D * 2 + ((c ^ (key & 7)) << 4));
        cp16(dst + at, static_cast<const uint16_t*>(a.k) + k0 + c * 8, full);
        cp16(dst + TILE + at, static_cast<const uint16_t*>(a.v) + v0 + c * 8, full);
      }
      ++fetched;
      if (fetched < total) {
        attn_next(a, pf);
        next_id = block_of(pf);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < AT_STAGES - 1; ++s) fetch();

  // ---- consumer -------------------------------------------------------------
  uint32_t qf[D / 16][4];
  float o[D / 8][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
  int lim0 = -1, lim1 = -1;  // last key that this lane's two query rows see
  const int g = lane >> 2, tq = lane & 3;
  bool fresh = true;
  for (int done = 0; done < total; ++done) {
    if (fresh) {  // a new item: its queries
      fresh = false;
      const int M = p.x.n * a.G;
      auto limit = [&](int row) {
        if (row >= M) return -1;
        return p.x.causal ? min(p.x.len - p.x.n + row / a.G, p.x.len - 1) : p.x.len - 1;
      };
      const int r0 = p.tile * AT_ROWS + g, r1 = r0 + 8;
      lim0 = limit(r0);
      lim1 = limit(r1);
      const uint16_t* base = static_cast<const uint16_t*>(a.q) + static_cast<int64_t>(p.h) * a.G * a.qh;
      const uint16_t* q0 = base + static_cast<int64_t>(p.x.t0 + r0 / a.G) * a.qt + (r0 % a.G) * a.qh + 2 * tq;
      const uint16_t* q1 = base + static_cast<int64_t>(p.x.t0 + r1 / a.G) * a.qt + (r1 % a.G) * a.qh + 2 * tq;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        qf[k][0] = r0 < M ? *reinterpret_cast<const uint32_t*>(q0 + 16 * k) : 0u;
        qf[k][1] = r1 < M ? *reinterpret_cast<const uint32_t*>(q1 + 16 * k) : 0u;
        qf[k][2] = r0 < M ? *reinterpret_cast<const uint32_t*>(q0 + 16 * k + 8) : 0u;
        qf[k][3] = r1 < M ? *reinterpret_cast<const uint32_t*>(q1 + 16 * k + 8) : 0u;
      }
#pragma unroll
      for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
      m0 = m1 = -INFINITY;
      l0 = l1 = 0.0f;
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(AT_STAGES - 2) : "memory");
    __syncwarp();
    fetch();  // into the stage that the last unit has left
    const uint32_t kt = ring + static_cast<uint32_t>((done % AT_STAGES) * 2 * TILE), vt = kt + TILE;

    float s[AT_KEYS / 8][4];
#pragma unroll
    for (int i = 0; i < AT_KEYS / 8; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
    {
      // lane -> row of the four 8x8 matrices: keys (lane & 7) + 8 * (lane >> 4), chunk + ((lane >> 3) & 1)
      const int kr = (lane & 7) + ((lane >> 4) << 3), cc = (lane >> 3) & 1;
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
#pragma unroll
        for (int n = 0; n < AT_KEYS / 16; ++n) {
          uint32_t b[4];
          const int key = n * 16 + kr;
          ldsm4(b, kt + static_cast<uint32_t>(key * D * 2 + (((2 * k + cc) ^ (key & 7)) << 4)));
          mma16816<BF16>(s[2 * n], qf[k], b[0], b[1]);
          mma16816<BF16>(s[2 * n + 1], qf[k], b[2], b[3]);
        }
    }
    const int j0 = p.u * AT_KEYS;
    const bool cut = j0 + AT_KEYS - 1 > min(lim0, lim1);
    float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
    for (int i = 0; i < AT_KEYS / 8; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        s[i][e] *= a.scale_log2;
        s[i][2 + e] *= a.scale_log2;
        if (cut) {
          const int j = j0 + 8 * i + 2 * tq + e;
          if (j > lim0) s[i][e] = -INFINITY;
          if (j > lim1) s[i][2 + e] = -INFINITY;
        }
        x0 = fmaxf(x0, s[i][e]);
        x1 = fmaxf(x1, s[i][2 + e]);
      }
    x0 = fmaxf(x0, __shfl_xor_sync(FULL, x0, 1));
    x1 = fmaxf(x1, __shfl_xor_sync(FULL, x1, 1));
    x0 = fmaxf(x0, __shfl_xor_sync(FULL, x0, 2));
    x1 = fmaxf(x1, __shfl_xor_sync(FULL, x1, 2));
    const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
    const float b0 = n0 == -INFINITY ? 0.0f : n0, b1 = n1 == -INFINITY ? 0.0f : n1;
    if (__any_sync(FULL, n0 != m0 || n1 != m1)) {
      const float c0 = ex2(m0 - b0), c1 = ex2(m1 - b1);  // 0 for the item's first unit (m = -inf)
      l0 *= c0;
      l1 *= c1;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        o[i][0] *= c0;
        o[i][1] *= c0;
        o[i][2] *= c1;
        o[i][3] *= c1;
      }
      m0 = n0;
      m1 = n1;
    }
    // p as the sum of two 16-bit values: rounding p to one would be the
    // largest error of a query that sees few keys, and the second product
    // with the same V fragments hides behind the loads
    uint32_t pr[AT_KEYS / 8][2], pl[AT_KEYS / 8][2];
#pragma unroll
    for (int i = 0; i < AT_KEYS / 8; ++i) {
      const float e0 = ex2(s[i][0] - b0), e1 = ex2(s[i][1] - b0), e2 = ex2(s[i][2] - b1), e3 = ex2(s[i][3] - b1);
      l0 += e0 + e1;
      l1 += e2 + e3;
      pr[i][0] = pack2<BF16>(e0, e1);
      pr[i][1] = pack2<BF16>(e2, e3);
      const float2 h0 = unpack2<BF16>(pr[i][0]), h1 = unpack2<BF16>(pr[i][1]);
      pl[i][0] = pack2<BF16>(e0 - h0.x, e1 - h0.y);
      pl[i][1] = pack2<BF16>(e2 - h1.x, e3 - h1.y);
    }
    {
      // keys (lane & 7) + 8 * ((lane >> 3) & 1), chunk + (lane >> 4)
      const int kr = (lane & 7) + (((lane >> 3) & 1) << 3), cc = lane >> 4;
#pragma unroll
      for (int n = 0; n < AT_KEYS / 16; ++n) {
        const uint32_t pa[4] = {pr[2 * n][0], pr[2 * n][1], pr[2 * n + 1][0], pr[2 * n + 1][1]};
        const uint32_t pb[4] = {pl[2 * n][0], pl[2 * n][1], pl[2 * n + 1][0], pl[2 * n + 1][1]};
        const int key = n * 16 + kr;
#pragma unroll
        for (int dd = 0; dd < D / 16; ++dd) {
          uint32_t b[4];
          ldsm4t(b, vt + static_cast<uint32_t>(key * D * 2 + (((2 * dd + cc) ^ (key & 7)) << 4)));
          mma16816<BF16>(o[2 * dd], pa, b[0], b[1]);
          mma16816<BF16>(o[2 * dd + 1], pa, b[2], b[3]);
          mma16816<BF16>(o[2 * dd], pb, b[0], b[1]);
          mma16816<BF16>(o[2 * dd + 1], pb, b[2], b[3]);
        }
      }
    }
    __syncwarp();  // every lane has read the stage before it is refilled

    const int item = p.item;
    const AttnPos was = p;
    if (done + 1 < total) attn_next(a, p);
    if (done + 1 == total || p.item != item) {  // the warp's part of this item is complete
      fresh = true;
      l0 += __shfl_xor_sync(FULL, l0, 1);
      l1 += __shfl_xor_sync(FULL, l1, 1);
      l0 += __shfl_xor_sync(FULL, l0, 2);
      l1 += __shfl_xor_sync(FULL, l1, 2);
      const long long slot = gw + item;
      const int M = was.x.n * a.G - was.tile * AT_ROWS;
      if (slot < a.slots) {
        float* po = a.part_o + slot * (AT_ROWS * D);
        if (g < M) {
#pragma unroll
          for (int i = 0; i < D / 8; ++i)
            *reinterpret_cast<float2*>(po + g * D + 8 * i + 2 * tq) = make_float2(o[i][0], o[i][1]);
          if (tq == 0) a.part_ml[slot * AT_ROWS + g] = make_float2(m0, l0);
        }
        if (g + 8 < M) {
#pragma unroll
          for (int i = 0; i < D / 8; ++i)
            *reinterpret_cast<float2*>(po + (g + 8) * D + 8 * i + 2 * tq) = make_float2(o[i][2], o[i][3]);
          if (tq == 0) a.part_ml[slot * AT_ROWS + g + 8] = make_float2(m1, l1);
        }
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  // this grid may have started beside the prefix kernel's: it does not end
  // before that one, so that the join, which waits for this grid, has both
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (bad_block && a.error_word) atomicOr(a.error_word, Q3S_DECERR_BLOCK_ID);
}

// Joins the parts of each query row (m, l, o as above) and writes out and lse.
// One warp a row; a lane holds D / 32 of its values and, for up to 32 parts at
// a time, one part's m and l.  Block (b, h, z): rows z, z + gridDim.z, ... of
// batch row b's n * G (times the block's warps); b == B: the tokens past the
// last row, which see nothing.
template <int D, bool BF16>
__global__ void __launch_bounds__(128) attn_join_kernel(const AttnArgs a) {
  constexpr int E = D / 32;
  const int w = static_cast<int>(threadIdx.x) >> 5, lane = static_cast<int>(threadIdx.x) & 31;
  const int b = static_cast<int>(blockIdx.x), h = static_cast<int>(blockIdx.y);
  AttnRow x;
  if (b < a.B) {
    x = attn_row(a, b + 1);
  } else {
    x.t0 = a.B ? min(max(a.offsets[a.B], 0), a.T) : 0;
    x.n = a.T - x.t0;
    x.units = x.tiles = 0;
  }
  const int M = x.n * a.G;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long* first = reinterpret_cast<const long long*>(a.plan);
  const int32_t* items = a.plan + 2 * (2 + a.B);
  const long long quota = first[0];
  for (int row = static_cast<int>(blockIdx.z) * 4 + w; row < M; row += static_cast<int>(gridDim.z) * 4) {
    const int token = x.t0 + row / a.G, gq = row % a.G;
    float acc[E], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
    // parts [0, n) at slots slot0 + i (or stride `step` rows apart), row `r` of each
    auto join = [&](const float* po, const float2* pml, int n, int64_t step) {
      for (int i0 = 0; i0 < n; i0 += 32) {
        const int k = min(n - i0, 32);
        float2 ml = make_float2(-INFINITY, 0.0f);
        if (lane < k) ml = pml[(i0 + lane) * step];
        float top = ml.x;
#pragma unroll
        for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, d));
        const float nm = fmaxf(m, top);
        if (nm == -INFINITY) continue;
        const float c = ex2(m - nm);
        m = nm;
        l *= c;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] *= c;
        const float wt = ex2(ml.x - nm);
        float lw = wt * ml.y;
#pragma unroll
        for (int d = 16; d; d >>= 1) lw += __shfl_xor_sync(FULL, lw, d);
        l += lw;
#pragma unroll 4
        for (int i = 0; i < k; ++i) {
          const float wi = __shfl_sync(FULL, wt, i);
          const float* src = po + (i0 + i) * step * D + lane * E;
          if constexpr (E == 4) {
            const float4 y = *reinterpret_cast<const float4*>(src);
            acc[0] += wi * y.x;
            acc[1] += wi * y.y;
            acc[2] += wi * y.z;
            acc[3] += wi * y.w;
          } else {
            const float2 y = *reinterpret_cast<const float2*>(src);
            acc[0] += wi * y.x;
            acc[1] += wi * y.y;
          }
        }
      }
    };
    // slots of an item: one a warp whose range meets the item's units
    auto join_item = [&](int r, const AttnRow& y, int tile) {
      const int in = h * y.tiles + tile;
      const long long us = first[1 + r] + static_cast<long long>(in) * y.units, ue = us + y.units - 1;
      const long long w0 = us / quota, w1 = ue / quota, slot = w0 + items[r] + in;
      if (w1 - w0 + slot >= a.slots) return;
      const int64_t at = slot * AT_ROWS;
      return join(a.part_o + (at + (r == 0 ? (token * a.G + gq) % AT_ROWS : row % AT_ROWS)) * D,
                  a.part_ml + at + (r == 0 ? (token * a.G + gq) % AT_ROWS : row % AT_ROWS),
                  static_cast<int>(w1 - w0) + 1, AT_ROWS);
    };
    if (a.prefix_here) {
      const AttnRow y = attn_row(a, 0);
      if (y.units) join_item(0, y, (token * a.G + gq) / AT_ROWS);
    } else if (a.splits) {
      const int64_t at = static_cast<int64_t>(token) * a.Hq + h * a.G + gq;
      join(a.pre_o + at * D, a.pre_ml + at, a.splits, static_cast<int64_t>(a.T) * a.Hq);
    }
    if (x.units) join_item(b + 1, x, row / AT_ROWS);
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    uint16_t* dst = static_cast<uint16_t*>(a.out) + token * a.ot + (h * a.G + gq) * a.oh + lane * E;
    if constexpr (E == 4)
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<BF16>(acc[0] * inv, acc[1] * inv), pack2<BF16>(acc[2] * inv, acc[3] * inv));
    else
      *reinterpret_cast<uint32_t*>(dst) = pack2<BF16>(acc[0] * inv, acc[1] * inv);
    if (a.lse && lane == 0)
      a.lse[static_cast<int64_t>(token) * a.Hq + h * a.G + gq] = l > 0.0f ? (m + log2f(l)) * 0.69314718055994531f : -INFINITY;
  }
}

}  // namespace q3s
