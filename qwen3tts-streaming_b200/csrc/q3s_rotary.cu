// q3s_rotary.cu -- rotary positions of queries and keys, with the append of
// keys and values to the paged cache (q3s_rotary).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "q3s_args.cuh"
#include "q3s_decode.h"
#include "q3s_device.cuh"
#include "q3s_pdl.cuh"

namespace q3s {

struct RotaryArgs {
  int T, Hq, Hk, dim, pairs, axes, bs, blocks;
  int sections[Q3S_MAX_ROTARY_AXES];
  bool interleaved;
  float scale;
  int turned, copied;  // units of a head that turn (pairs of vectors with HALF) and that are only copied
  const int32_t* positions;
  int64_t position_stride;
  const float* inv_freq;
  const void *q, *k, *v;
  void *out, *kc, *vc;
  int64_t qt, qh, ot, oh, kt, kh, vt, vh, kb, kch, kp, vb, vch, vp;
  const int64_t* slots;
  int32_t* error_word;
};

constexpr int RO_MAX_NT = 256;
constexpr int RO_ANGLES = 512;  // cos and sin that a CTA holds: its tokens times the pairs
constexpr int RO_TOKENS = 4;    // the most tokens of a CTA

// cos and sin of pos * freq.  The product is taken in 64 bits, in turns (off by
// 3 * 2^-53 of the angle: 7e-7 of a radian at an angle of 2^31), where whole
// quarters come off it exactly; what is left, at most an eighth of a turn, is
// rounded to 32 bits once (2^-24 of it, 5e-8 of a radian).
Q3S_DEV float2 rotary_angle(int pos, float freq, float scale) {
  const double turns = static_cast<double>(pos) * (static_cast<double>(freq) * 0.15915494309189533577);  // 1 / (2 pi)
  const double quarters = rint(turns * 4.0);
  const float left = static_cast<float>(2.0 * (turns - quarters * 0.25));  // in half turns
  float s, c;
  sincospif(left, &s, &c);
  const int quadrant = static_cast<int>(static_cast<long long>(quarters) & 3);
  const float x = quadrant & 1 ? s : c, y = quadrant & 1 ? c : s;
  return make_float2((quadrant == 1 || quadrant == 2 ? -x : x) * scale, (quadrant >= 2 ? -y : y) * scale);
}

// Two neighbouring values, converted together: single conversions to or from 16 bits go through
// the unit of the transcendental functions, a quarter as fast (8191 tokens 39 us).
Q3S_DEV float2 to_f32(const float* x) { return make_float2(x[0], x[1]); }
Q3S_DEV float2 to_f32(const __nv_bfloat16* x) {
  const uint32_t w = *reinterpret_cast<const uint32_t*>(x);
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
Q3S_DEV float2 to_f32(const __half* x) { return __half22float2(*reinterpret_cast<const __half2*>(x)); }
Q3S_DEV void from_f32(float* x, float2 f) { x[0] = f.x, x[1] = f.y; }
Q3S_DEV void from_f32(__nv_bfloat16* x, float2 f) { *reinterpret_cast<__nv_bfloat162*>(x) = __floats2bfloat162_rn(f.x, f.y); }
Q3S_DEV void from_f32(__half* x, float2 f) { *reinterpret_cast<__half2*>(x) = __floats2half2_rn(f.x, f.y); }

template <typename T, int E>
struct alignas(sizeof(T) * E) RotaryVec {
  T x[E];
};

// One head row's unit u.  A unit that turns is two vectors of E elements, E of
// the pairs (HALF), or one vector of E / 2 neighbouring pairs; at E = 1 the
// neighbours are two units of one element, taken as HALF is.
template <typename T, int E, bool ADJ>
struct RotaryUnit {
  using Vec = RotaryVec<T, E>;
  static constexpr bool TWO = !ADJ || E == 1;
  Vec a, b;
  Q3S_DEV static int first(int u, int turned) { return u < turned ? (ADJ ? (E == 1 ? 2 * u : u * E) : u * E) : 0; }
  Q3S_DEV void load(const T* from, int u, int turned, int pairs) {
    if (u < turned) {
      const int at = first(u, turned);
      a = *reinterpret_cast<const Vec*>(from + at);
      if constexpr (TWO) b = *reinterpret_cast<const Vec*>(from + at + (ADJ ? 1 : pairs));
    } else {
      a = *reinterpret_cast<const Vec*>(from + 2 * pairs + (u - turned) * E);
    }
  }
  // cs: cos and sin of the token's pairs
  Q3S_DEV void turn(const float2* cs, int u, int turned) {
    if (u >= turned) return;
    // pair i of a unit is at i * units, so that neighbouring lanes read neighbouring places
    if constexpr (E == 1) {
      const float2 c = cs[u];
      float p = static_cast<float>(a.x[0]), q = static_cast<float>(b.x[0]);
      one(c, p, q);
      a.x[0] = static_cast<T>(p), b.x[0] = static_cast<T>(q);
    } else if constexpr (TWO) {
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        float2 p = to_f32(a.x + e), q = to_f32(b.x + e);
        one(cs[u + e * turned], p.x, q.x);
        one(cs[u + (e + 1) * turned], p.y, q.y);
        from_f32(a.x + e, p), from_f32(b.x + e, q);
      }
    } else {
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        float2 p = to_f32(a.x + 2 * e);
        one(cs[u + e * turned], p.x, p.y);
        from_f32(a.x + 2 * e, p);
      }
    }
  }
  static constexpr int PAIRS = TWO ? E : E / 2;  // of a unit
  Q3S_DEV static void one(float2 c, float& x, float& y) {
    const float p = x, q = y;
    x = fmaf(p, c.x, -(q * c.y));
    y = fmaf(p, c.y, q * c.x);
  }
  Q3S_DEV void store(T* to, int u, int turned, int pairs) const {
    if (u < turned) {
      const int at = first(u, turned);
      *reinterpret_cast<Vec*>(to + at) = a;
      if constexpr (TWO) *reinterpret_cast<Vec*>(to + at + (ADJ ? 1 : pairs)) = b;
    } else {
      *reinterpret_cast<Vec*>(to + 2 * pairs + (u - turned) * E) = a;
    }
  }
};

// A CTA takes up to four neighbouring tokens and one share of their heads
// (blockIdx.y); a thread keeps a unit of a head (two 16-byte vectors) for all of
// them, so that addresses are counted up and not divided out (one unit after another of
// tokens times heads took 39 us for 8191 tokens, bound by instructions).  The units of queries or keys and of values are requested before
// anything else; while they are on their way the threads compute the cos and sin of the
// tokens' pairs, one each, into shared memory, where all heads find them.  Bound by HBM: every byte is read and written
// once; 8191 tokens of 16 and 8 heads of 128 in 16 bits, 133 MB, take 26.8 us, 5.0 TB/s (6.55 a copy), the rest being
// the latency of a CTA's one round of loads at 33 % of the warps.  (64 registers in place of 78, for four CTAs a SM: spills, 32.7 us.)
template <typename T, int E, bool ADJ>
__global__ void __launch_bounds__(RO_MAX_NT) rotary_kernel(const RotaryArgs a, int tokens) {
  using Unit = RotaryUnit<T, E, ADJ>;
  using Vec = RotaryVec<T, E>;
  __shared__ float2 s_cs[RO_ANGLES];
  __shared__ int64_t s_k[RO_TOKENS], s_v[RO_TOKENS];  // offsets of a token's place in the caches; -1: none
  const int t = static_cast<int>(threadIdx.x), nt = static_cast<int>(blockDim.x);
  const int first = static_cast<int>(blockIdx.y) * nt + t, all = static_cast<int>(gridDim.y) * nt;  // of a unit a thread
  const int64_t token0 = static_cast<int64_t>(blockIdx.x) * tokens;
  const int n = static_cast<int>(min(static_cast<int64_t>(tokens), a.T - token0));
  const int units = a.turned + a.copied, items = (a.Hq + a.Hk) * units, vunits = a.dim / E, vitems = a.Hk * vunits;
  grid_wait();
  grid_release();

  Unit x[RO_TOKENS];
  Vec y[RO_TOKENS];
  auto fetch = [&](int item) {
    const int h = item / units, u = item - h * units;
    const bool query = h < a.Hq;
    const T* from = query ? static_cast<const T*>(a.q) + token0 * a.qt + h * a.qh : static_cast<const T*>(a.k) + token0 * a.kt + (h - a.Hq) * a.kh;
    const int64_t stride = query ? a.qt : a.kt;
#pragma unroll
    for (int i = 0; i < RO_TOKENS; ++i)
      if (i < n) x[i].load(from + i * stride, u, a.turned, a.pairs);
  };
  auto finish = [&](int item) {
    const int h = item / units, u = item - h * units;
    const bool query = h < a.Hq;
    T* to = query ? static_cast<T*>(a.out) + token0 * a.ot + h * a.oh : static_cast<T*>(a.kc) + (h - a.Hq) * a.kch;
#pragma unroll
    for (int i = 0; i < RO_TOKENS; ++i) {
      if (i >= n || (!query && s_k[i] < 0)) continue;
      x[i].turn(s_cs + i * a.pairs, u, a.turned);
      x[i].store(to + (query ? i * a.ot : s_k[i]), u, a.turned, a.pairs);
    }
  };
  auto fetch_v = [&](int item) {  // values are copied whole
    const int h = item / vunits, u = item - h * vunits;
    const T* from = static_cast<const T*>(a.v) + token0 * a.vt + h * a.vh + u * E;
#pragma unroll
    for (int i = 0; i < RO_TOKENS; ++i)
      if (i < n) y[i] = *reinterpret_cast<const Vec*>(from + i * a.vt);
  };
  auto finish_v = [&](int item) {
    const int h = item / vunits, u = item - h * vunits;
    T* to = static_cast<T*>(a.vc) + h * a.vch + u * E;
#pragma unroll
    for (int i = 0; i < RO_TOKENS; ++i)
      if (i < n && s_v[i] >= 0) *reinterpret_cast<Vec*>(to + s_v[i]) = y[i];
  };
  if (first < items) fetch(first);
  if (first < vitems) fetch_v(first);

  for (int i = t; i < n * a.pairs; i += nt) {
    const int tok = i / a.pairs, p = i - tok * a.pairs;
    int axis = 0;
    if (a.axes > 1) {
      if (a.interleaved) {
        const int m = p % a.axes;
        axis = p < a.axes * a.sections[m] ? m : 0;
      } else {
        int end = a.sections[0];
        while (p >= end && axis + 1 < a.axes) end += a.sections[++axis];
      }
    }
    s_cs[tok * a.pairs + p / Unit::PAIRS + p % Unit::PAIRS * a.turned] = rotary_angle(a.positions[axis * a.position_stride + token0 + tok], a.inv_freq[p], a.scale);
  }
  if (a.Hk && nt - 1 - t < n) {  // the last threads, which have the fewest angles
    const int i = nt - 1 - t;
    const int64_t slot = a.slots[token0 + i];
    s_k[i] = s_v[i] = -1;
    if (slot >= static_cast<int64_t>(a.blocks) * a.bs) {
      if (a.error_word && blockIdx.y == 0) atomicOr(a.error_word, Q3S_DECERR_BLOCK_ID);
    } else if (slot >= 0) {
      const int64_t block = (slot >> 32) == 0 ? static_cast<int64_t>(static_cast<uint32_t>(slot) / static_cast<uint32_t>(a.bs)) : slot / a.bs;
      const int64_t place = slot - block * a.bs;
      s_k[i] = block * a.kb + place * a.kp;
      s_v[i] = block * a.vb + place * a.vp;
    }
  }
  __syncthreads();
  for (int item = first; item < items; item += all) {
    if (item != first) fetch(item);
    finish(item);
  }
  for (int item = first; item < vitems; item += all) {
    if (item != first) fetch_v(item);
    finish_v(item);
  }
}

template <typename T, int E, bool ADJ>
cudaError_t launch_rotary(RotaryArgs a, cudaStream_t st) {
  // units of a head: two vectors, or one where the neighbours are in it
  const int turned = !ADJ || E == 1 ? a.pairs / E : 2 * a.pairs / E;
  a.turned = turned;
  a.copied = (a.dim - 2 * a.pairs) / E;
  // Threads: a unit each, up to 256 (more units: several in turn).
  const int64_t items = std::max<int64_t>(static_cast<int64_t>(a.Hq + a.Hk) * (turned + a.copied), static_cast<int64_t>(a.Hk) * (a.dim / E));
  const int nt = static_cast<int>(std::min<int64_t>((items + 31) / 32 * 32, RO_MAX_NT));
  // Tokens a CTA: up to four (and what its angles have room for) while there are four CTAs a SM.  Up to four
  // against up to two: 8191 tokens of 16 and 8 heads of 128 in 16 bits 26.8 and
  // 28.0 us, 5000 of 12 heads of 80 in 32 bits 11.1 and 12.4.
  const int sms = sm_count();
  const int tokens = std::max(std::min(std::min(RO_ANGLES / a.pairs, RO_TOKENS), a.T / (4 * sms)), 1);
  // shares of the units while there are fewer CTAs than SMs
  const int64_t ctas = (static_cast<int64_t>(a.T) + tokens - 1) / tokens;
  const int64_t shares = std::max<int64_t>(std::min<int64_t>(std::min<int64_t>((items + nt - 1) / nt, sms / ctas), 65535), 1);
  return launch_maybe_pdl(rotary_kernel<T, E, ADJ>, dim3(static_cast<unsigned>(ctas), static_cast<unsigned>(shares)), dim3(nt), 0, st, true, a,
                          tokens);
}

template <typename T>
cudaError_t launch_rotary(const RotaryArgs& a, bool vec, bool adjacent, cudaStream_t st) {
  constexpr int E = 16 / sizeof(T);
  return vec ? (adjacent ? launch_rotary<T, E, true>(a, st) : launch_rotary<T, E, false>(a, st))
             : (adjacent ? launch_rotary<T, 1, true>(a, st) : launch_rotary<T, 1, false>(a, st));
}

}  // namespace q3s

extern "C" q3s_status q3s_rotary(const q3s_rotary_desc* d, void* stream) {
  using q3s::report;
  if (!d) return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_rotary: desc is NULL");
  if (d->struct_size != sizeof(q3s_rotary_desc))
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_rotary: struct_size %u != %u (ABI mismatch)", d->struct_size,
                  static_cast<unsigned>(sizeof(q3s_rotary_desc)));
  if (d->tokens < 0 || d->q_heads < 0 || d->kv_heads < 0 || d->dim < 2)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_rotary: tokens, q_heads and kv_heads must not be negative and dim at least 2");
  if ((static_cast<int64_t>(d->q_heads) + d->kv_heads) * d->dim > (1 << 24))
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_rotary: heads * dim is above 2^24");
  if (d->pairs < 1 || d->pairs > d->dim / 2)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_rotary: %d pairs of %d elements", d->pairs, d->dim);
  if (d->pairs > q3s::RO_ANGLES)
    return report(Q3S_ERR_UNSUPPORTED, "q3s_rotary: %d pairs are more than %d", d->pairs, q3s::RO_ANGLES);
  if (d->flags & ~(Q3S_ROTARY_ADJACENT | Q3S_ROTARY_INTERLEAVED))
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_rotary: unknown flags %#x", d->flags);
  if (d->elem != Q3S_ELEM_F32 && d->elem != Q3S_ELEM_BF16 && d->elem != Q3S_ELEM_F16)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_rotary: unknown elem %d", d->elem);
  if (d->axes < 1 || d->axes > Q3S_MAX_ROTARY_AXES)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_rotary: %d axes are not 1 to %d", d->axes, Q3S_MAX_ROTARY_AXES);
  int64_t total = 0;
  for (int i = 0; i < d->axes; ++i) {
    if (d->sections[i] < 0) return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_rotary: section %d is negative", i);
    total += d->sections[i];
    // the last place of axis i > 0, axes * (section - 1) + i, is a pair
    if ((d->flags & Q3S_ROTARY_INTERLEAVED) && i > 0 && d->sections[i] > 0 &&
        static_cast<int64_t>(d->axes) * (d->sections[i] - 1) + i >= d->pairs)
      return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_rotary: section %d of %d has no room between %d interleaved pairs", i,
                    d->sections[i], d->pairs);
  }
  if (total != d->pairs)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_rotary: sections of %lld pairs in all, not %d", static_cast<long long>(total), d->pairs);
  if (d->kv_heads > 0 && (d->block_size < 1 || d->blocks < 1))
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_rotary: block_size and blocks must be positive");
  if (d->tokens == 0 || d->q_heads + d->kv_heads == 0) return report(Q3S_OK, "");
  if (!d->positions || !d->inv_freq) return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_rotary: positions and inv_freq are required");
  if (d->q_heads > 0 && (!d->q || !d->out)) return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_rotary: q and out are required");
  if (d->q == d->out && d->q_heads > 0 && (d->q_token_stride != d->out_token_stride || d->q_head_stride != d->out_head_stride))
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_rotary: q and out in place must have the same strides");
  if (d->kv_heads > 0 && (!d->k || !d->v || !d->slot_map || !d->k_cache || !d->v_cache))
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_rotary: k, v, slot_map, k_cache and v_cache are required");
  q3s::RotaryArgs a;
  a.T = d->tokens;
  a.Hq = d->q_heads;
  a.Hk = d->kv_heads;
  a.dim = d->dim;
  a.pairs = d->pairs;
  a.axes = d->axes;
  a.bs = d->block_size;
  a.blocks = d->blocks;
  for (int i = 0; i < Q3S_MAX_ROTARY_AXES; ++i) a.sections[i] = i < d->axes ? d->sections[i] : 0;
  a.interleaved = (d->flags & Q3S_ROTARY_INTERLEAVED) != 0;
  a.scale = d->scale;
  a.positions = d->positions;
  a.position_stride = d->position_stride;
  a.inv_freq = d->inv_freq;
  a.q = d->q;
  a.out = d->out;
  a.k = d->k;
  a.v = d->v;
  a.kc = d->k_cache;
  a.vc = d->v_cache;
  a.qt = d->q_token_stride;
  a.qh = d->q_head_stride;
  a.ot = d->out_token_stride;
  a.oh = d->out_head_stride;
  a.kt = d->k_token_stride;
  a.kh = d->k_head_stride;
  a.vt = d->v_token_stride;
  a.vh = d->v_head_stride;
  a.kb = d->k_block_stride;
  a.kch = d->k_cache_head_stride;
  a.kp = d->k_place_stride;
  a.vb = d->v_block_stride;
  a.vch = d->v_cache_head_stride;
  a.vp = d->v_place_stride;
  a.slots = d->slot_map;
  a.error_word = d->error_word;
  // 16-byte vectors where every base, stride and cut of a head allows them, single elements otherwise
  const bool adjacent = (d->flags & Q3S_ROTARY_ADJACENT) != 0;
  const int64_t e = d->elem == Q3S_ELEM_F32 ? 4 : 8;
  bool vec = d->dim % e == 0 && (adjacent ? 2 * d->pairs : d->pairs) % e == 0;
  if (d->q_heads > 0) {
    for (int64_t x : {a.qt, a.qh, a.ot, a.oh}) vec = vec && x % e == 0;
    for (const void* p : {d->q, static_cast<const void*>(d->out)}) vec = vec && (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
  }
  if (d->kv_heads > 0) {
    for (int64_t x : {a.kt, a.kh, a.vt, a.vh, a.kb, a.kch, a.kp, a.vb, a.vch, a.vp}) vec = vec && x % e == 0;
    for (const void* p : {d->k, d->v, static_cast<const void*>(d->k_cache), static_cast<const void*>(d->v_cache)})
      vec = vec && (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
  }
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t err = d->elem == Q3S_ELEM_F32    ? q3s::launch_rotary<float>(a, vec, adjacent, st)
                          : d->elem == Q3S_ELEM_BF16 ? q3s::launch_rotary<__nv_bfloat16>(a, vec, adjacent, st)
                                                     : q3s::launch_rotary<__half>(a, vec, adjacent, st);
  if (err != cudaSuccess) return report(Q3S_ERR_CUDA, "q3s_rotary: launch failed: %s", cudaGetErrorString(err));
  return report(Q3S_OK, "");
}
