// q3s_int8.cuh -- 8-bit projections: per-row quantisation and the matrix
// product with a scale per row and per output channel.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "q3s_args.cuh"
#include "q3s_decode.h"
#include "q3s_device.cuh"
#include "q3s_head.cuh"

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
// few.  VEC = false: bases, strides or K that 16-byte accesses cannot take.
template <int ELEM, bool VEC>
__global__ void __launch_bounds__(128) quantize_rows_kernel(const QuantArgs a) {
  using E = Elem<ELEM>;
  constexpr int NT = 128, KEEP = 4, N = E::N;
  __shared__ float s_red[NT / 32];
  const int t = static_cast<int>(threadIdx.x);
  asm volatile("griddepcontrol.launch_dependents;");
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

// ---- the matrix product -------------------------------------------------------

struct Int8Args {
  int M, N, K;
  int mtiles, ntiles, kchunks;
  const float* a_scales;
  const float* w_scales;
  const float* bias;
  void* y;
  int64_t ldy;
  bool vec_y;  // 16-byte stores of y are aligned
  int32_t* error_word;
};

Q3S_DEV void umma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}

constexpr int I8_BM = 128;   // rows of a tile: the matrix instruction's M
constexpr int I8_BK = 128;   // bytes of a row in one 128-byte swizzled chunk
constexpr int I8_NT = 192;   // 4 epilogue warps, the copy warp, the matrix warp
constexpr int I8_A_BYTES = I8_BM * I8_BK;

template <int BN>
struct I8Tile {
  static constexpr int STAGE = I8_A_BYTES + BN * I8_BK;
  static constexpr int STAGES = (200 * 1024) / STAGE < 8 ? (200 * 1024) / STAGE : 8;
  static constexpr int SMEM = 1024 + STAGES * STAGE + 256;
  static constexpr int TMEM = 2 * BN < 32 ? 32 : 2 * BN;  // two accumulators
  // kind::i8: 32-bit integer accumulator (2), A and B signed (1), both
  // K-major, N >> 3 in [17, 23), M >> 4 in [24, 29)
  static constexpr uint32_t IDESC = (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(BN >> 3) << 17) |
                                    (static_cast<uint32_t>(I8_BM >> 4) << 24);
};

// Persistent tiles of 128 x BN: one warp copies (TMA, 128-byte swizzle), one
// issues the matrix instructions (one elected thread), four scale and store
// the previous tile out of the other half of TMEM meanwhile.  The sums are
// exact 32-bit integers (K <= 131072 keeps them below 2^31), so their order
// does not matter; each output is rounded once. 
template <int BN, int ELEM>
__global__ void __launch_bounds__(I8_NT, 1)
    int8_matmul_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_w,
                       const Int8Args a) {
  using Tile = I8Tile<BN>;
  using E = Elem<ELEM>;
  constexpr int STAGES = Tile::STAGES;
  extern __shared__ __align__(1024) unsigned char i8_smem[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(i8_smem) + 1023) &
                                                         ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * Tile::STAGE);
  uint64_t* empty = full + STAGES;
  uint64_t* ready = empty + STAGES;  // [2] an accumulator is complete
  uint64_t* drained = ready + 2;     // [2] an accumulator has been read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 2);
  int* failed = reinterpret_cast<int*>(tmem_slot + 1);
  const int t = static_cast<int>(threadIdx.x), w = t >> 5, lane = t & 31;
  const int tiles = a.mtiles * a.ntiles;

  if (t == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&ready[b], 1);
      mbar_init(&drained[b], 128);
    }
    *failed = 0;
    fence_mbar_init();
  }
  if (w == 5) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(Tile::TMEM)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the quantised rows, when this grid is launched behind them

  // a wait that gives up marks the CTA; every role then stops at its next wait
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (*reinterpret_cast<volatile int*>(failed)) return false;
    if (mbar_wait_bounded(bar, parity)) return true;
    atomicOr(failed, 1);
    return false;
  };

  if (w == 4) {
    if (lane == 0) {
      int k = 0;  // chunks so far
      bool ok = true;
      for (int tile = static_cast<int>(blockIdx.x); ok && tile < tiles; tile += static_cast<int>(gridDim.x)) {
        const int m0 = (tile % a.mtiles) * I8_BM, n0 = (tile / a.mtiles) * BN;
        for (int c = 0; c < a.kchunks; ++c, ++k) {
          const int s = k % STAGES;
          if (k >= STAGES && !wait(&empty[s], ((k / STAGES) - 1) & 1)) {
            ok = false;
            break;
          }
          unsigned char* st = smem + s * Tile::STAGE;
          mbar_expect_tx(&full[s], Tile::STAGE);
          tma_load_2d(smem_u32(st), &tm_a, c * I8_BK, m0, &full[s]);
          tma_load_2d(smem_u32(st + I8_A_BYTES), &tm_w, c * I8_BK, n0, &full[s]);
        }
      }
      // no copy may be in flight when the CTA leaves: wait for each stage's last one
      for (int i = max(0, k - STAGES); i < k; ++i) (void)mbar_wait_bounded(&full[i % STAGES], (i / STAGES) & 1);
    }
  } else if (w == 5) {
    if (lane == 0) {
      int k = 0, i = 0;
      bool ok = true;
      for (int tile = static_cast<int>(blockIdx.x); ok && tile < tiles; tile += static_cast<int>(gridDim.x), ++i) {
        const int b = i & 1;
        if (i >= 2 && !wait(&drained[b], ((i >> 1) - 1) & 1)) break;
        tc_fence_after();
        for (int c = 0; c < a.kchunks; ++c, ++k) {
          const int s = k % STAGES;
          if (!wait(&full[s], (k / STAGES) & 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + s * Tile::STAGE);
          const uint64_t da = head_smem_desc(sa), db = head_smem_desc(sa + I8_A_BYTES);
#pragma unroll
          for (int j = 0; j < I8_BK / 32; ++j)  // 32 bytes of K = 2 descriptor units per instruction
            umma_i8(tmem + static_cast<uint32_t>(b * BN), da + 2 * j, db + 2 * j, Tile::IDESC, (c | j) != 0);
          umma_commit(&empty[s]);
        }
        umma_commit(&ready[b]);
      }
    }
  } else {
    int i = 0;
    for (int tile = static_cast<int>(blockIdx.x); tile < tiles; tile += static_cast<int>(gridDim.x), ++i) {
      const int b = i & 1;
      const int n0 = (tile / a.mtiles) * BN, row = (tile % a.mtiles) * I8_BM + 32 * w + lane;
      const bool in = row < a.M;
      const float as = in ? a.a_scales[row] : 0.0f;
      if (!__all_sync(FULL, wait(&ready[b], (i >> 1) & 1))) break;
      tc_fence_after();
      typename E::T* y = static_cast<typename E::T*>(a.y) + row * a.ldy + n0;
#pragma unroll 1
      for (int c = 0; c < BN / 32; ++c) {
        float v[32];
        tmem_ld32(tmem + (static_cast<uint32_t>(32 * w) << 16) + static_cast<uint32_t>(b * BN + 32 * c), v);
        if (n0 + 32 * c >= a.N) continue;
        const int left = a.N - n0 - 32 * c;
        if (left >= 32 && a.vec_y) {
          const float* ws = a.w_scales + n0 + 32 * c;
          const float* bi = a.bias ? a.bias + n0 + 32 * c : nullptr;
#pragma unroll
          for (int j = 0; j < 32; ++j)
            v[j] = __fmul_rn(__fmul_rn(static_cast<float>(__float_as_int(v[j])), as), __ldg(ws + j));
          if (bi) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] += __ldg(bi + j);
          }
          if (in) {
            constexpr int W = 16 / sizeof(typename E::T);
#pragma unroll
            for (int j = 0; j < 32; j += W) {
              typename E::T p[W];
#pragma unroll
              for (int q = 0; q < W; ++q) p[q] = E::narrow(v[j + q]);
              uint4 u;
              memcpy(&u, p, 16);
              *reinterpret_cast<uint4*>(y + 32 * c + j) = u;
            }
          }
        } else if (in) {
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            if (j >= left) break;
            float x = __fmul_rn(__fmul_rn(static_cast<float>(__float_as_int(v[j])), as), a.w_scales[n0 + 32 * c + j]);
            if (a.bias) x += a.bias[n0 + 32 * c + j];
            y[32 * c + j] = E::narrow(x);
          }
        }
      }
      tc_fence_before();
      asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&drained[b])) : "memory");
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (w == 5) {
    tc_fence_after();
    if (*failed) {  // matrix instructions may still be running: their commits (bounded) before the columns go
      if (lane == 0)
        for (int b = 0; b < 2; ++b) (void)mbar_wait_bounded(&ready[b], 0);
      __syncwarp();
    }
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Tile::TMEM) : "memory");
  }
  if (t == 0 && *failed && a.error_word) atomicOr(a.error_word, Q3S_DECERR_WAIT);
}

}  // namespace q3s
