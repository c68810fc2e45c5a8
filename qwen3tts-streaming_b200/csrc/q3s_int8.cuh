// q3s_int8.cuh -- 8-bit projections: per-row quantisation and the matrix
// product with a scale per row and per output channel.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

#include "q3s_args.cuh"
#include "q3s_decode.h"
#include "q3s_device.cuh"
#include "q3s_head.cuh"
#include "q3s_pdl.cuh"

namespace q3s {

// ---- element types ----------------------------------------------------------
// 16 bytes of x as fp32: 8 values of a 2-byte type, 4 of fp32.
template <int ELEM>
struct Elem;
template <>
struct Elem<Q3S_ELEM_F32> {
  using T = float;
  static constexpr int N = 4;
  Q3S_DEV static void widen(const uint4& u, float (&x)[N]) {
    x[0] = __uint_as_float(u.x);
    x[1] = __uint_as_float(u.y);
    x[2] = __uint_as_float(u.z);
    x[3] = __uint_as_float(u.w);
  }
  Q3S_DEV static float one(const T* p) { return *p; }
  Q3S_DEV static T narrow(float x) { return x; }
  Q3S_DEV static uint32_t narrow2(const float* x) { return __float_as_uint(x[0]); }  // 32 bits of output
};
template <>
struct Elem<Q3S_ELEM_BF16> {
  using T = uint16_t;
  static constexpr int N = 8;
  Q3S_DEV static void widen(const uint4& u, float (&x)[N]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  Q3S_DEV static float one(const T* p) { return __uint_as_float(static_cast<uint32_t>(*p) << 16); }
  Q3S_DEV static T narrow(float x) {
    uint16_t r;
    asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(r) : "f"(x));
    return r;
  }
  Q3S_DEV static uint32_t narrow2(const float* x) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(x[1]), "f"(x[0]));
    return r;
  }
};
template <>
struct Elem<Q3S_ELEM_F16> {
  using T = uint16_t;
  static constexpr int N = 8;
  Q3S_DEV static float half(uint16_t h) {
    float f;
    asm("cvt.f32.f16 %0, %1;" : "=f"(f) : "h"(h));
    return f;
  }
  Q3S_DEV static void widen(const uint4& u, float (&x)[N]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = half(static_cast<uint16_t>(w[i] & 0xffffu));
      x[2 * i + 1] = half(static_cast<uint16_t>(w[i] >> 16));
    }
  }
  Q3S_DEV static float one(const T* p) { return half(*p); }
  Q3S_DEV static T narrow(float x) {
    uint16_t r;
    asm("cvt.rn.f16.f32 %0, %1;" : "=h"(r) : "f"(x));
    return r;
  }
  Q3S_DEV static uint32_t narrow2(const float* x) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(x[1]), "f"(x[0]));
    return r;
  }
};

// ---- quantisation -----------------------------------------------------------

constexpr float QUANT_TINY = 7.888609052210118e-31f;  // 2^-100

// Largest magnitude of two, NaN if either is.
Q3S_DEV float absmax(float m, float x) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(x)));
  return r;
}
struct QuantScale {
  float scale, unit;  // a / 127 and 127 / a
};
Q3S_DEV QuantScale quant_scale(float a) {
  if (!(a <= 3.4028234663852886e38f)) return {__int_as_float(0x7fffffff), 0.0f};  // infinity or NaN
  if (a < QUANT_TINY) return {0.0f, 0.0f};                                         // 127 / a might overflow
  return {__fdiv_rn(a, 127.0f), __fdiv_rn(127.0f, a)};
}
// Nearest even; |x * unit| <= 127 (1 + 2^-23), which rounds to 127 at most.
// An infinity or NaN comes with unit 0: its product is NaN, which converts to 0.
Q3S_DEV int quant_one(float x, float unit) { return __float2int_rn(__fmul_rn(x, unit)); }

struct QuantArgs {
  int M, K;
  const void* x;
  int64_t ldx;
  int8_t* values;
  int64_t ldv;
  float* scales;
};

// Block-wide maximum over NT threads (NaN if any thread's is).
template <int NT>
Q3S_DEV float block_absmax(float m, float* s_red) {
#pragma unroll
  for (int d = 16; d; d >>= 1) m = absmax(m, __shfl_xor_sync(FULL, m, d));
  if ((threadIdx.x & 31) == 0) s_red[threadIdx.x >> 5] = m;
  __syncthreads();
  m = s_red[0];
#pragma unroll
  for (int i = 1; i < NT / 32; ++i) m = absmax(m, s_red[i]);
  return m;
}

// One CTA a row: one pass over the row for its largest magnitude, the values
// kept in registers (KEEP 16-byte loads a thread; what is beyond them is read
// again, from L2) for the second.  Bound by HBM for many rows, by latency for
// few: 130 rows of 2048 1.7 us.  VEC = false: bases, strides or K that 16-byte
// accesses cannot take.
template <int ELEM, bool VEC>
__global__ void __launch_bounds__(128) quantize_rows_kernel(const QuantArgs a) {
  using E = Elem<ELEM>;
  constexpr int NT = 128, KEEP = 4, N = E::N;
  __shared__ float s_red[NT / 32];
  const int t = static_cast<int>(threadIdx.x);
  grid_wait();
  grid_release();
  const int64_t row = blockIdx.x;
  const typename E::T* x = static_cast<const typename E::T*>(a.x) + row * a.ldx;
  int8_t* out = a.values + row * a.ldv;
  float m = 0.0f;
  if constexpr (VEC) {
    const int chunks = a.K / N;
    uint4 keep[KEEP];
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
      const int c = t + NT * i;
      keep[i] = c < chunks ? ld_stream16(x + static_cast<int64_t>(c) * N) : make_uint4(0, 0, 0, 0);
    }
    float v[N];
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
      E::widen(keep[i], v);
#pragma unroll
      for (int j = 0; j < N; ++j) m = absmax(m, v[j]);
    }
    for (int c = t + NT * KEEP; c < chunks; c += NT) {
      E::widen(*reinterpret_cast<const uint4*>(x + static_cast<int64_t>(c) * N), v);
#pragma unroll
      for (int j = 0; j < N; ++j) m = absmax(m, v[j]);
    }
    const QuantScale s = quant_scale(block_absmax<NT>(m, s_red));
    auto store = [&](int c, const uint4& u) {
      E::widen(u, v);
      uint32_t p[N / 4];
#pragma unroll
      for (int j = 0; j < N / 4; ++j) {
        uint32_t w = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b) w |= (static_cast<uint32_t>(quant_one(v[4 * j + b], s.unit)) & 0xffu) << (8 * b);
        p[j] = w;
      }
      if constexpr (N == 8)
        *reinterpret_cast<uint2*>(out + static_cast<int64_t>(c) * N) = make_uint2(p[0], p[1]);
      else
        *reinterpret_cast<uint32_t*>(out + static_cast<int64_t>(c) * N) = p[0];
    };
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
      if (t + NT * i < chunks) store(t + NT * i, keep[i]);
    for (int c = t + NT * KEEP; c < chunks; c += NT)
      store(c, *reinterpret_cast<const uint4*>(x + static_cast<int64_t>(c) * N));
    if (t == 0) a.scales[row] = s.scale;
  } else {
    for (int c = t; c < a.K; c += NT) m = absmax(m, E::one(x + c));
    const QuantScale s = quant_scale(block_absmax<NT>(m, s_red));
    for (int c = t; c < a.K; c += NT) out[c] = static_cast<int8_t>(quant_one(E::one(x + c), s.unit));
    if (t == 0) a.scales[row] = s.scale;
  }
}

// Many rows of up to 256 sixteen-byte units: a warp a row, the whole row in
// registers, all its loads in flight at once and no barrier.  8192 rows of 2048
// (50 MB): 11.9 us from cold, 4.2 TB/s.  Four warps a CTA: with eight 4096 rows of
// 2048 took 4.6 us against 4.4; more CTAs a SM spill (5.4).
constexpr int QW_WARPS = 4, QW_KEEP = 8;
template <int ELEM>
__global__ void __launch_bounds__(QW_WARPS * 32) quantize_warps_kernel(const QuantArgs a) {
  using E = Elem<ELEM>;
  constexpr int N = E::N;
  grid_wait();
  grid_release();
  const int lane = static_cast<int>(threadIdx.x) & 31, chunks = a.K / N;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * QW_WARPS + (threadIdx.x >> 5);
  if (row >= a.M) return;
  const typename E::T* x = static_cast<const typename E::T*>(a.x) + row * a.ldx;
  uint4 keep[QW_KEEP];
#pragma unroll
  for (int i = 0; i < QW_KEEP; ++i)
    keep[i] = lane + 32 * i < chunks ? ld_stream16(x + static_cast<int64_t>(lane + 32 * i) * N) : make_uint4(0, 0, 0, 0);
  float v[N], m = 0.0f;
#pragma unroll
  for (int i = 0; i < QW_KEEP; ++i) {
    E::widen(keep[i], v);
#pragma unroll
    for (int j = 0; j < N; ++j) m = absmax(m, v[j]);
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) m = absmax(m, __shfl_xor_sync(FULL, m, d));
  const QuantScale s = quant_scale(m);
  if (lane == 0) a.scales[row] = s.scale;
  int8_t* out = a.values + row * a.ldv;
#pragma unroll
  for (int i = 0; i < QW_KEEP; ++i) {
    if (lane + 32 * i >= chunks) break;
    E::widen(keep[i], v);
    uint32_t p[N / 4];
#pragma unroll
    for (int j = 0; j < N / 4; ++j) {
      p[j] = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b) p[j] |= (static_cast<uint32_t>(quant_one(v[4 * j + b], s.unit)) & 0xffu) << (8 * b);
    }
    if constexpr (N == 8)
      *reinterpret_cast<uint2*>(out + (lane + 32 * i) * N) = make_uint2(p[0], p[1]);
    else
      *reinterpret_cast<uint32_t*>(out + (lane + 32 * i) * N) = p[0];
  }
}

// ---- the matrix product -------------------------------------------------------

struct Int8Args {
  int M, N, K;
  const int8_t* a;
  int64_t lda;
  const float* a_scales;
  const int8_t* w;
  int64_t ldw;
  const float* w_scales;
  const float* bias;
  void* y;
  int64_t ldy;
  bool vec_y;  // 16-byte accesses of y's rows are aligned
  int32_t* error_word;
};

// An output from its exact sum.
Q3S_DEV float int8_out(int sum, float a_scale, float w_scale) {
  return __fmul_rn(__fmul_rn(static_cast<float>(sum), a_scale), w_scale);
}

// -- few rows: one pass over the weights with 8-bit dot products -----------------

constexpr int GV_NT = 256, GV_WARPS = GV_NT / 32;
constexpr int GV_MAX_M = 8;
constexpr int GV_SMEM = 24 * 1024;  // most bytes of activations

// M <= MB <= 8 rows: the product is bound by reading the weights once, and at
// these sizes by latency.  A warp owns RW outputs and reads their weight rows
// 512 bytes at a time, the first rounds of all of them before anything else
// (after the grid's wait: the weights may come from the kernel before); the
// activations sit in shared memory as bytes; sums are reduced over the warp by
// one integer instruction each.  QUANT: the rows of x are quantised here, by
// every CTA for itself (they are few), with the weights already on their way,
// so a Linear is one launch; CTA 0 writes the values and scales out.  1 x 2048 x
// 2048 (4.2 MB): 2.5 us a launch, weights from L2; 1 x 2048 x 8000 4.0 us, 4.1 TB/s.
template <bool QUANT, int ELEM, int MB, int RW>
__global__ void __launch_bounds__(GV_NT) int8_gemv_kernel(const Int8Args a, const QuantArgs q) {
  using E = Elem<ELEM>;
  constexpr int AHEAD = 4;  // rounds of 512 bytes of each row requested at the start
  extern __shared__ __align__(16) unsigned char gv_smem[];  // [MB][K] activations
  __shared__ float s_max[GV_WARPS], s_scale[MB];
  const int t = static_cast<int>(threadIdx.x), w = t >> 5, lane = t & 31;
  const int n0 = (static_cast<int>(blockIdx.x) * GV_WARPS + w) * RW;
  const int rounds = (a.K + 511) / 512;
  grid_wait();
  grid_release();
  uint4 first[RW][AHEAD];
#pragma unroll
  for (int r = 0; r < RW; ++r)
#pragma unroll
    for (int c = 0; c < AHEAD; ++c) {
      const int k = 512 * c + 16 * lane;
      first[r][c] = n0 + r < a.N && k < a.K ? ld_stream16(a.w + (n0 + r) * a.ldw + k) : make_uint4(0, 0, 0, 0);
    }
  if constexpr (QUANT) {
    constexpr int GROUP = GV_NT / MB, KEEP = 4;  // threads of a row; 16-byte loads that stay in registers
    const int m = t / GROUP, i = t % GROUP, chunks = a.K / E::N;
    const typename E::T* x = static_cast<const typename E::T*>(q.x) + m * q.ldx;
    uint4 keep[KEEP];
    float v[E::N], top = 0.0f;
#pragma unroll
    for (int c = 0; c < KEEP; ++c)
      keep[c] = m < a.M && i + GROUP * c < chunks
                    ? *reinterpret_cast<const uint4*>(x + static_cast<int64_t>(i + GROUP * c) * E::N)
                    : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int c = 0; c < KEEP; ++c) {
      E::widen(keep[c], v);
#pragma unroll
      for (int j = 0; j < E::N; ++j) top = absmax(top, v[j]);
    }
    if (m < a.M)
      for (int c = i + GROUP * KEEP; c < chunks; c += GROUP) {
        E::widen(*reinterpret_cast<const uint4*>(x + static_cast<int64_t>(c) * E::N), v);
#pragma unroll
        for (int j = 0; j < E::N; ++j) top = absmax(top, v[j]);
      }
#pragma unroll
    for (int d = 16; d; d >>= 1) top = absmax(top, __shfl_xor_sync(FULL, top, d));
    if (lane == 0) s_max[w] = top;
    __syncthreads();
    constexpr int WR = GROUP / 32;  // warps of a row
    top = s_max[(w / WR) * WR];
#pragma unroll
    for (int j = 1; j < WR; ++j) top = absmax(top, s_max[(w / WR) * WR + j]);
    const QuantScale s = quant_scale(top);
    const bool out = blockIdx.x == 0 && m < a.M;
    if (i == 0) {
      s_scale[m] = s.scale;
      if (out) q.scales[m] = s.scale;
    }
    auto store = [&](int c, const uint4& u) {
      E::widen(u, v);
      uint32_t p[E::N / 4];
#pragma unroll
      for (int j = 0; j < E::N / 4; ++j) {
        p[j] = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b) p[j] |= (static_cast<uint32_t>(quant_one(v[4 * j + b], s.unit)) & 0xffu) << (8 * b);
      }
      uint32_t* dst = reinterpret_cast<uint32_t*>(gv_smem + static_cast<size_t>(m) * a.K + static_cast<size_t>(c) * E::N);
      uint32_t* copy = reinterpret_cast<uint32_t*>(q.values + m * q.ldv + static_cast<int64_t>(c) * E::N);
#pragma unroll
      for (int j = 0; j < E::N / 4; ++j) {
        dst[j] = p[j];
        if (out) copy[j] = p[j];
      }
    };
#pragma unroll
    for (int c = 0; c < KEEP; ++c)
      if (i + GROUP * c < chunks) store(i + GROUP * c, keep[c]);
    for (int c = i + GROUP * KEEP; c < chunks; c += GROUP)
      store(c, m < a.M ? *reinterpret_cast<const uint4*>(x + static_cast<int64_t>(c) * E::N) : make_uint4(0, 0, 0, 0));
  } else {
    for (int c = t; c < MB * (a.K / 16); c += GV_NT) {
      const int m = c / (a.K / 16), k = 16 * (c - m * (a.K / 16));
      reinterpret_cast<uint4*>(gv_smem)[c] = m < a.M ? *reinterpret_cast<const uint4*>(a.a + m * a.lda + k) : make_uint4(0, 0, 0, 0);
    }
    if (t < MB) s_scale[t] = t < a.M ? a.a_scales[t] : 0.0f;
  }
  __syncthreads();

  int acc[RW][MB];
#pragma unroll
  for (int r = 0; r < RW; ++r)
#pragma unroll
    for (int m = 0; m < MB; ++m) acc[r][m] = 0;
  auto round = [&](int k, const uint4 (&wv)[RW]) {  // 16 bytes of K a lane
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      const uint4 x = *reinterpret_cast<const uint4*>(gv_smem + static_cast<size_t>(m) * a.K + k);
#pragma unroll
      for (int r = 0; r < RW; ++r) {
        acc[r][m] = __dp4a(static_cast<int>(wv[r].x), static_cast<int>(x.x), acc[r][m]);
        acc[r][m] = __dp4a(static_cast<int>(wv[r].y), static_cast<int>(x.y), acc[r][m]);
        acc[r][m] = __dp4a(static_cast<int>(wv[r].z), static_cast<int>(x.z), acc[r][m]);
        acc[r][m] = __dp4a(static_cast<int>(wv[r].w), static_cast<int>(x.w), acc[r][m]);
      }
    }
  };
#pragma unroll
  for (int c = 0; c < AHEAD; ++c) {
    uint4 wv[RW];
#pragma unroll
    for (int r = 0; r < RW; ++r) wv[r] = first[r][c];
    if (512 * c + 16 * lane < a.K) round(512 * c + 16 * lane, wv);
  }
#pragma unroll 2
  for (int c = AHEAD; c < rounds; ++c) {
    const int k = 512 * c + 16 * lane;
    if (k >= a.K) break;
    uint4 wv[RW];
#pragma unroll
    for (int r = 0; r < RW; ++r) wv[r] = n0 + r < a.N ? ld_stream16(a.w + (n0 + r) * a.ldw + k) : make_uint4(0, 0, 0, 0);
    round(k, wv);
  }
  __syncwarp();
  int mine = 0;  // lane r * MB + m: that sum
#pragma unroll
  for (int r = 0; r < RW; ++r)
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      const int sum = __reduce_add_sync(FULL, acc[r][m]);
      if (lane == r * MB + m) mine = sum;
    }
  const int m = lane % MB, n = n0 + lane / MB;
  if (lane < RW * MB && m < a.M && n < a.N) {
    float v = int8_out(mine, s_scale[m], a.w_scales[n]);
    if (a.bias) v += a.bias[n];
    static_cast<typename E::T*>(a.y)[m * a.ldy + n] = E::narrow(v);
  }
}

// -- tensor cores -----------------------------------------------------------------

constexpr int I8_BK = 128;   // bytes of a row in one 128-byte swizzled chunk
constexpr int I8_TILE = 128 * I8_BK;  // 128 rows of a chunk

// kind::i8: 32-bit integer accumulator (2), A and B signed (1), both K-major,
// N >> 3 in [17, 23), M >> 4 in [24, 29).
__host__ __device__ constexpr uint32_t i8_idesc(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
Q3S_DEV void umma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}
Q3S_DEV void umma_i8_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}
// Arrive on `bar` of both CTAs of the pair once the products issued before are complete.
Q3S_DEV void umma_commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}
// A copy into this CTA's shared memory that completes on the barrier at
// shared::cluster address `bar` (the pair's leading CTA).
Q3S_DEV void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::
          "r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
Q3S_DEV void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
Q3S_DEV void tma_store_2d(const CUtensorMap* map, int x, int y, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(src)
               : "memory");
}
Q3S_DEV void cluster_arrive_release() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
Q3S_DEV int4 ld_cluster16(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

// Up to a few hundred rows: the weights are the matrix instruction's M (128
// outputs a CTA), the rows of x its N (BT, a multiple of 32), so that one pass
// over the weights serves all rows of a tile; K is cut over the KS CTAs of a
// cluster so that all SMs read.  The partial sums (32-bit integers, exact in any
// order) meet in distributed shared memory: CTA r of a cluster finishes every
// KS-th group of tokens.  Bound by the latency of that chain (load, products,
// exchange) and the weights' bytes: 130 x 2048 x 5000 takes 7.8 us after the
// quantisation's 1.7 (12 MB, 1.9 us at HBM's rate).
struct I8Cut {
  int bt, stages, chunks;  // tokens of a tile, ring stages, chunks of K
  int tmem;                // columns: a power of two >= 32
  int ks, smem;            // CTAs of a cluster, dynamic shared memory
};
constexpr int I8C_NT = 256;

inline I8Cut int8_cut(int M, int N, int K, int sms) {
  I8Cut cut;
  cut.chunks = (K + I8_BK - 1) / I8_BK;
  const int ntiles = (N + 127) / 128;
  // Tile height and K cut: the lowest estimate of the time in clocks.  A CTA loads
  // its operands (168 bytes a clock of a SM, shared by the CTAs there), reads its
  // sums out of TMEM and joins its share of the cluster's; two CTAs share a SM
  // where three stages of each fit, and overlap all but a little of the latter.
  // The constants are fitted to 400 timings over 26 shapes from 12 x 2048 x 5000
  // to 8000 x 512 x 100, on which the choice is 3% slower than the best in the
  // mean and 12% at most.
  auto stage_of = [](int bt) { return I8_TILE + bt * I8_BK; };
  auto per_sm = [&](int bt) { return 110 * 1024 / stage_of(bt) >= 3 && bt * 512 <= 108 * 1024 ? 2 : 1; };
  const double cluster_clocks[4] = {0, 50, 730, 2350};  // of 1, 2, 4, 8 CTAs
  cut.ks = 1;
  double best = 0;
  for (int mt = (M + 255) / 256; mt <= (M + 31) / 32; ++mt) {
    const int bt = ((M + mt - 1) / mt + 31) / 32 * 32;
    if ((M + bt - 1) / bt != mt) continue;
    for (int e = 0; e < 4 && cut.chunks >= (1 << e); ++e) {
      const int k = 1 << e;
      const double ctas = static_cast<double>(ntiles) * mt * k;
      const double waves = std::ceil(ctas / (per_sm(bt) * sms)), share = waves > 1 ? per_sm(bt) : std::max(1.0, ctas / sms);
      const double loads = static_cast<double>((cut.chunks + k - 1) / k) * stage_of(bt) / 168;
      const double sums = 2.6 * bt + cluster_clocks[e] + 24.0 * bt / k;
      const double cost = waves * (loads * share + sums * (1 + 0.06 * (share - 1)));
      if (best == 0 || cost < best) {
        best = cost;
        cut.bt = bt;
        cut.ks = k;
      }
    }
  }
  const int mtiles = (M + cut.bt - 1) / cut.bt, stage = stage_of(cut.bt);
  cut.tmem = 32;
  while (cut.tmem < cut.bt) cut.tmem *= 2;
  const bool two = static_cast<int64_t>(ntiles) * mtiles * cut.ks > sms && per_sm(cut.bt) == 2;
  const int mine = (cut.chunks + cut.ks - 1) / cut.ks;
  // a ring that also holds the partial sums of the tile
  const int least = (cut.bt * 512 + stage - 1) / stage;
  cut.stages = std::max(least, std::min({8, mine, (two ? 110 : 196) * 1024 / stage}));
  cut.smem = std::max(1024 + cut.stages * stage, TMEM_PART_SMEM);
  return cut;
}

template <int ELEM, int KS>
__global__ void __launch_bounds__(I8C_NT)
    int8_split_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_a, const Int8Args a,
                      const I8Cut cut) {
  using E = Elem<ELEM>;
  extern __shared__ __align__(1024) unsigned char i8_smem[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(i8_smem) + 1023) &
                                                         ~static_cast<uintptr_t>(1023));
  __shared__ __align__(8) uint64_t full[8], empty[8], ready;
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  const int t = static_cast<int>(threadIdx.x), w = t >> 5, lane = t & 31;
  const int n0 = static_cast<int>(blockIdx.x) * 128, rank = static_cast<int>(cluster_rank());
  const int token0 = static_cast<int>(blockIdx.z) * cut.bt;
  const int stage_bytes = I8_TILE + cut.bt * I8_BK;
  const int c0 = cut.chunks * rank / KS, count = cut.chunks * (rank + 1) / KS - c0;  // this CTA's chunks, >= 1
  if (t == 0) {
    for (int s = 0; s < cut.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&ready, 1);
    failed = 0;
    fence_mbar_init();
  }
  if (w == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(cut.tmem)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  if (t == 0) {
    grid_wait();  // rows and weights may both come from the kernel before
    for (int c = 0; c < count; ++c) {
      const int s = c % cut.stages;
      if (c >= cut.stages && !mbar_wait_bounded(&empty[s], ((c / cut.stages) - 1) & 1)) {
        atomicOr(&failed, 1);
        break;
      }
      const uint32_t dst = smem_u32(smem + s * stage_bytes);
      mbar_expect_tx(&full[s], stage_bytes);
      tma_load_2d(dst, &tm_w, (c0 + c) * I8_BK, n0, &full[s]);
      tma_load_2d(dst + I8_TILE, &tm_a, (c0 + c) * I8_BK, token0, &full[s]);
    }
  } else if (t == 32) {
    const uint32_t idesc = i8_idesc(128, cut.bt);
    for (int c = 0; c < count; ++c) {
      const int s = c % cut.stages;
      if (!mbar_wait_bounded(&full[s], (c / cut.stages) & 1)) {
        atomicOr(&failed, 1);
        break;
      }
      tc_fence_after();
      const uint32_t sa = smem_u32(smem + s * stage_bytes);
      const uint64_t dw = head_smem_desc(sa), da = head_smem_desc(sa + I8_TILE);
#pragma unroll
      for (int j = 0; j < I8_BK / 32; ++j)  // 32 bytes of K = 2 descriptor units per instruction
        umma_i8(tmem, dw + 2 * j, da + 2 * j, idesc, (c | j) != 0);
      umma_commit(&empty[s]);
    }
    umma_commit(&ready);
  }
  __syncwarp();
  grid_wait();
  grid_release();
  const bool done = mbar_wait_bounded(&ready, 0);
  if (!done) atomicOr(&failed, 1);
  tc_fence_after();
  // every product is complete: the ring holds the partial sums now, [token][128
  // outputs]; warp w reads TMEM lanes 32 (w % 4) .., every other 32 columns
  int* part = reinterpret_cast<int*>(smem);
  for (int c = 32 * (w >> 2); c < cut.bt; c += 64) {
    float v[32];
    tmem_ld32(tmem + (static_cast<uint32_t>(32 * (w & 3)) << 16) + static_cast<uint32_t>(c), v);
#pragma unroll
    for (int i = 0; i < 32; ++i) part[(c + i) * 128 + (t & 127)] = __float_as_int(v[i]);
  }
  tc_fence_before();
  cluster_arrive_release();
  cluster_wait();  // every CTA's partial sums are in place
  {
    const int n = n0 + 4 * lane;
    float ws[4], bi[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      ws[j] = n + j < a.N ? a.w_scales[n + j] : 0.0f;
      bi[j] = a.bias && n + j < a.N ? a.bias[n + j] : 0.0f;
    }
    constexpr int T = KS == 8 ? 2 : 4, STEP = KS * (I8C_NT / 32);  // tokens of a warp in flight, and their distance
    for (int tok0 = rank * (I8C_NT / 32) + w; tok0 < cut.bt && token0 + tok0 < a.M; tok0 += T * STEP) {
      int4 part_sum[T][KS];
#pragma unroll
      for (int i = 0; i < T; ++i) {
        const int tok = min(tok0 + i * STEP, cut.bt - 1);
#pragma unroll
        for (int k = 0; k < KS; ++k) part_sum[i][k] = ld_cluster16(cluster_addr(smem_u32(part + tok * 128 + 4 * lane), k));
      }
#pragma unroll
      for (int i = 0; i < T; ++i) {
        const int tok = tok0 + i * STEP;
        if (tok >= cut.bt || token0 + tok >= a.M) break;
        int4 sum = part_sum[i][0];
#pragma unroll
        for (int k = 1; k < KS; ++k) {
          sum.x += part_sum[i][k].x;
          sum.y += part_sum[i][k].y;
          sum.z += part_sum[i][k].z;
          sum.w += part_sum[i][k].w;
        }
        const float as = a.a_scales[token0 + tok];
        const float v[4] = {int8_out(sum.x, as, ws[0]) + bi[0], int8_out(sum.y, as, ws[1]) + bi[1],
                            int8_out(sum.z, as, ws[2]) + bi[2], int8_out(sum.w, as, ws[3]) + bi[3]};
        typename E::T* y = static_cast<typename E::T*>(a.y) + static_cast<int64_t>(token0 + tok) * a.ldy + n;
        if (a.vec_y && n + 4 <= a.N) {
          typename E::T o[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) o[j] = E::narrow(v[j]);
          if constexpr (sizeof(o) == 8) *reinterpret_cast<uint2*>(y) = *reinterpret_cast<uint2*>(o);
          else *reinterpret_cast<uint4*>(y) = *reinterpret_cast<uint4*>(o);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n + j < a.N) y[j] = E::narrow(v[j]);
        }
      }
    }
  }
  cluster_arrive_relaxed();
  cluster_wait();  // nobody leaves while its sums are being read
  if (failed && t == 0) {  // copies and products still in flight, bounded
    for (int s = 0; s < cut.stages && s < count; ++s) (void)mbar_wait_bounded(&full[s], 0);
    (void)mbar_wait_bounded(&ready, 0);
    if (a.error_word) atomicOr(a.error_word, Q3S_DECERR_WAIT);
  }
  __syncthreads();
  if (w == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cut.tmem) : "memory");
  }
}

// Many rows: persistent 256 x 256 tiles, one a pair of CTAs (cta_group::2: each
// holds 128 rows of x and 128 of the weights, the instruction reads both
// halves), because at 8 bits the operands of a one-CTA instruction would take
// more than the shared memory gives and twice the L2 reads (128 x 128 tiles of
// one CTA: 200 us for 8192 x 2048 x 8192; 128 x 256: 131 us; this: 98 us, 2.8
// POP/s, 72% of the tensor pipe; bursts of a few ms, 115 us in seconds of them,
// where the power limit takes the SMs to 1.47 GHz).  Bound by the products at the
// power limit, and at small K by the epilogue (79 us without one; 140 with 4-byte stores from
// registers, where a sixth stage changed nothing).  Per CTA: a copy warp, the
// leading CTA's matrix warp, and eight warps that scale and store the previous
// tile out of the other half of TMEM, through shared memory and TMA stores.
constexpr int I8P_EPI = 8, I8P_NT = (I8P_EPI + 2) * 32, I8P_STAGES = 5, I8P_N = 256;
constexpr int I8P_STAGE = 2 * I8_TILE;
constexpr int I8P_OUT = 4096;  // 32 rows of 128 bytes
constexpr int I8P_SMEM = 1024 + I8P_STAGES * I8P_STAGE + I8P_EPI * I8P_OUT + I8P_EPI * I8P_N * 4;
static_assert(I8P_SMEM >= TMEM_ALL_SMEM, "takes all of the tensor memory");

template <int ELEM>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(I8P_NT, 1)
    int8_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_w,
                     const __grid_constant__ CUtensorMap tm_y, const Int8Args a) {
  using E = Elem<ELEM>;
  constexpr int OC = 128 / static_cast<int>(sizeof(typename E::T));  // output columns in 128 bytes
  extern __shared__ __align__(1024) unsigned char i8_smem[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(i8_smem) + 1023) &
                                                         ~static_cast<uintptr_t>(1023));
  __shared__ __align__(8) uint64_t full[I8P_STAGES], empty[I8P_STAGES], ready[2], drained[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  const int t = static_cast<int>(threadIdx.x), w = t >> 5, lane = t & 31;
  const int rank = static_cast<int>(cluster_rank()), pairs = static_cast<int>(gridDim.x) / 2, pair = static_cast<int>(blockIdx.x) / 2;
  const int mtiles = (a.M + 255) / 256, tiles = mtiles * ((a.N + I8P_N - 1) / I8P_N), chunks = (a.K + I8_BK - 1) / I8_BK;
  if (t == 0) {
    for (int s = 0; s < I8P_STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&ready[b], 1);
      mbar_init(&drained[b], 2 * I8P_EPI);  // the epilogue warps of both CTAs
    }
    failed = 0;
    fence_mbar_init();
  }
  if (w == I8P_EPI + 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_arrive_release();
  cluster_wait();  // the pair's barriers are initialised and its TMEM is allocated
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  grid_wait();  // the quantised rows, when this grid is launched behind them
  grid_release();

  // a wait that gives up marks the CTA; every role then stops at its next wait
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*static_cast<volatile int*>(&failed)) return false;
    if (mbar_wait_bounded(bar, parity)) return true;
    atomicOr(&failed, 1);
    return false;
  };

  if (w == I8P_EPI) {
    if (lane == 0) {
      int k = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < tiles; tile += pairs) {
        const int m0 = (tile % mtiles) * 256 + 128 * rank, n0 = (tile / mtiles) * I8P_N + 128 * rank;
        for (int c = 0; c < chunks; ++c, ++k) {
          const int s = k % I8P_STAGES;
          if (k >= I8P_STAGES && !wait(&empty[s], ((k / I8P_STAGES) - 1) & 1)) {
            ok = false;
            break;
          }
          const uint32_t dst = smem_u32(smem + s * I8P_STAGE), bar = cluster_addr(smem_u32(&full[s]), 0);
          if (rank == 0) mbar_expect_tx(&full[s], 2 * I8P_STAGE);  // both CTAs' copies
          tma_load_2d_pair(dst, &tm_a, c * I8_BK, m0, bar);
          tma_load_2d_pair(dst + I8_TILE, &tm_w, c * I8_BK, n0, bar);
        }
      }
      // no copy may be in flight when the pair leaves: the stages' last ones (they complete on the leading CTA)
      if (rank == 0)
        for (int i = max(0, k - I8P_STAGES); i < k; ++i) (void)mbar_wait_bounded(&full[i % I8P_STAGES], (i / I8P_STAGES) & 1);
    }
  } else if (w == I8P_EPI + 1) {
    if (rank == 0 && lane == 0) {
      constexpr uint32_t idesc = i8_idesc(256, I8P_N);
      int k = 0, i = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < tiles; tile += pairs, ++i) {
        const int b = i & 1;
        if (i >= 2 && !wait(&drained[b], ((i >> 1) - 1) & 1)) break;
        tc_fence_after();
        for (int c = 0; c < chunks; ++c, ++k) {
          const int s = k % I8P_STAGES;
          if (!wait(&full[s], (k / I8P_STAGES) & 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + s * I8P_STAGE);
          const uint64_t da = head_smem_desc(sa), dw = head_smem_desc(sa + I8_TILE);
#pragma unroll
          for (int j = 0; j < I8_BK / 32; ++j)  // 32 bytes of K = 2 descriptor units per instruction
            umma_i8_pair(tmem + static_cast<uint32_t>(b * I8P_N), da + 2 * j, dw + 2 * j, idesc, (c | j) != 0);
          umma_commit_pair(&empty[s]);
        }
        umma_commit_pair(&ready[b]);
      }
    }
  } else {
    // warp w: TMEM lanes (rows) 32 (w % 4) .., columns HALF (w / 4) ..
    constexpr int HALF = I8P_N / 2;
    unsigned char* buf = smem + I8P_STAGES * I8P_STAGE + w * I8P_OUT;
    float* s_ws = reinterpret_cast<float*>(smem + I8P_STAGES * I8P_STAGE + I8P_EPI * I8P_OUT) + w * 2 * HALF;  // scales, bias
    const int quarter = 32 * (w & 3), half = HALF * (w >> 2);
    int i = 0;
    for (int tile = pair; tile < tiles; tile += pairs, ++i) {
      const int b = i & 1, n0 = (tile / mtiles) * I8P_N + half, row0 = (tile % mtiles) * 256 + 128 * rank + quarter, row = row0 + lane;
      const float as = row < a.M ? a.a_scales[row] : 0.0f;
#pragma unroll
      for (int j = 0; j < HALF / 32; ++j) {
        const int n = n0 + 32 * j + lane;
        s_ws[32 * j + lane] = n < a.N ? a.w_scales[n] : 0.0f;
        if (a.bias) s_ws[HALF + 32 * j + lane] = n < a.N ? a.bias[n] : 0.0f;
      }
      __syncwarp();
      if (!__all_sync(FULL, wait(&ready[b], (i >> 1) & 1))) break;
      tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < HALF / OC; ++c) {
        uint32_t o[32];  // 128 bytes of the row
#pragma unroll
        for (int hc = 0; hc < OC / 32; ++hc) {
          float v[32];
          tmem_ld32(tmem + (static_cast<uint32_t>(quarter) << 16) + static_cast<uint32_t>(b * I8P_N + half + OC * c + 32 * hc), v);
          const float* ws = s_ws + OC * c + 32 * hc;
          const float2 as2 = make_float2(as, as);
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 s4 = *reinterpret_cast<const float4*>(ws + j);
            float2 x0 = make_float2(static_cast<float>(__float_as_int(v[j])), static_cast<float>(__float_as_int(v[j + 1])));
            float2 x1 = make_float2(static_cast<float>(__float_as_int(v[j + 2])), static_cast<float>(__float_as_int(v[j + 3])));
            x0 = __fmul2_rn(__fmul2_rn(x0, as2), make_float2(s4.x, s4.y));
            x1 = __fmul2_rn(__fmul2_rn(x1, as2), make_float2(s4.z, s4.w));
            v[j] = x0.x, v[j + 1] = x0.y, v[j + 2] = x1.x, v[j + 3] = x1.y;
          }
          if (a.bias) {
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              const float4 b4 = *reinterpret_cast<const float4*>(ws + HALF + j);
              v[j] += b4.x, v[j + 1] += b4.y, v[j + 2] += b4.z, v[j + 3] += b4.w;
            }
          }
#pragma unroll
          for (int j = 0; j < 32; j += 4 / static_cast<int>(sizeof(typename E::T)))
            o[(32 * hc + j) * static_cast<int>(sizeof(typename E::T)) / 4] = E::narrow2(v + j);
        }
        const int n = n0 + OC * c;
        if (c == HALF / OC - 1) {  // the accumulator has been read
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(cluster_addr(smem_u32(&drained[b]), 0));
        }
        if (n >= a.N || row0 >= a.M) continue;
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // the last store has left the buffer
        __syncwarp();
#pragma unroll
        for (int q = 0; q < 8; ++q)
          *reinterpret_cast<uint4*>(buf + lane * 128 + ((q ^ (lane & 7)) << 4)) =
              make_uint4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
        if (a.vec_y) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&tm_y, n, row0, smem_u32(buf));
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        } else {  // rows that do not start on 16 bytes: element by element, a row at a time
          __syncwarp();
          typename E::T* y = static_cast<typename E::T*>(a.y) + static_cast<int64_t>(row0) * a.ldy + n;
          const int rows = min(a.M - row0, 32);
#pragma unroll 4
          for (int r = 0; r < rows; ++r, y += a.ldy)
#pragma unroll
            for (int j = lane; j < OC; j += 32) {
              const int at = j * static_cast<int>(sizeof(typename E::T));
              if (n + j < a.N)
                y[j] = *reinterpret_cast<const typename E::T*>(buf + r * 128 + (((at >> 4) ^ (r & 7)) << 4) + (at & 15));
            }
          __syncwarp();
        }
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_arrive_release();
  cluster_wait();  // both CTAs are done with each other's barriers, shared memory and TMEM
  if (w == I8P_EPI + 1) {
    tc_fence_after();
    if (failed && rank == 0) {  // products may still be running: their commits (bounded) before the columns go
      if (lane == 0)
        for (int b = 0; b < 2; ++b) (void)mbar_wait_bounded(&ready[b], 0);
      __syncwarp();
    }
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
  if (t == 0 && failed && a.error_word) atomicOr(a.error_word, Q3S_DECERR_WAIT);
}

}  // namespace q3s
