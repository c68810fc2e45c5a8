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
  int per;             // head rows that a pass of the CTA takes
  const int32_t* positions;
  int64_t position_stride;
  const float* inv_freq;
  const void *q, *k, *v;
  void *out, *kc, *vc;
  int64_t qt, qh, ot, oh, kt, kh, vt, vh, kb, kch, kp, vb, vch, vp;
  const int64_t* slots;
  int32_t* error_word;
};

constexpr int RO_NT = 256;
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

template <typename T>
Q3S_DEV float to_f32(T x) {
  return static_cast<float>(x);
}
template <typename T>
Q3S_DEV T from_f32(float x) {
  return static_cast<T>(x);  // to nearest even
}

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
    if constexpr (TWO) {
#pragma unroll
      for (int e = 0; e < E; ++e) one(cs[u * E + e], a.x[e], b.x[e]);
    } else {
#pragma unroll
      for (int e = 0; e < E / 2; ++e) one(cs[u * (E / 2) + e], a.x[2 * e], a.x[2 * e + 1]);
    }
  }
  Q3S_DEV static void one(float2 c, T& x, T& y) {
    const float p = to_f32(x), q = to_f32(y);
    x = from_f32<T>(fmaf(p, c.x, -(q * c.y)));
    y = from_f32<T>(fmaf(p, c.y, q * c.x));
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

// A CTA takes TT tokens and one share of their heads (blockIdx.y).  Its threads
// first compute the cos and sin of the tokens' pairs, one each, into shared memory:
// all heads share them, and one evaluation a thread is the shortest way to the first
// store.  Then a thread keeps its unit of a head row (two 16-byte vectors) and
// walks the rows, queries, keys and values after one another, two at a time so that
// four to six loads are on their way.  Bound by HBM: every byte is read and written once.
template <typename T, int E, bool ADJ>
__global__ void __launch_bounds__(RO_NT) rotary_kernel(const RotaryArgs a, int tokens) {
  using Unit = RotaryUnit<T, E, ADJ>;
  __shared__ float2 s_cs[RO_ANGLES];
  __shared__ int64_t s_k[RO_TOKENS], s_v[RO_TOKENS];  // offsets of a token's place in the caches; -1: none
  const int t = static_cast<int>(threadIdx.x);
  const int64_t token0 = static_cast<int64_t>(blockIdx.x) * tokens;
  const int n = static_cast<int>(min(static_cast<int64_t>(tokens), a.T - token0));
  grid_wait();
  grid_release();
  for (int i = t; i < n * a.pairs; i += RO_NT) {
    const int tok = i / a.pairs, p = i - tok * a.pairs;
    int axis = 0;
    if (a.interleaved) {
      const int m = p % a.axes;
      axis = p < a.axes * a.sections[m] ? m : 0;
    } else {
      int end = a.sections[0];
      while (p >= end && axis + 1 < a.axes) end += a.sections[++axis];
    }
    s_cs[i] = rotary_angle(a.positions[axis * a.position_stride + token0 + tok], a.inv_freq[p], a.scale);
  }
  if (a.Hk)
    for (int i = t; i < n; i += RO_NT) {
      const int64_t slot = a.slots[token0 + i];
      s_k[i] = s_v[i] = -1;
      if (slot >= static_cast<int64_t>(a.blocks) * a.bs) {
        if (a.error_word && blockIdx.y == 0) atomicOr(a.error_word, Q3S_DECERR_BLOCK_ID);
      } else if (slot >= 0) {
        const int64_t block = slot / a.bs, place = slot - block * a.bs;
        s_k[i] = block * a.kb + place * a.kp;
        s_v[i] = block * a.vb + place * a.vp;
      }
    }
  __syncthreads();
  const int units = a.turned + a.copied, per = a.per;
  {
    const int row0 = t / units, first = t - row0 * units;
    const int heads = a.Hq + a.Hk, rows = n * heads, step = per * static_cast<int>(gridDim.y);
    if (row0 < per)
      for (int u = first; u < units; u += RO_NT)
        for (int r = static_cast<int>(blockIdx.y) * per + row0; r < rows; r += 2 * step) {
          Unit x[2];
          T* to[2];
          int tok[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int at = r + i * step;
            to[i] = nullptr;
            if (at >= rows) continue;
            tok[i] = at / heads;
            const int h = at - tok[i] * heads;
            const int64_t token = token0 + tok[i];
            const T* from;
            if (h < a.Hq) {
              from = static_cast<const T*>(a.q) + token * a.qt + h * a.qh;
              to[i] = static_cast<T*>(a.out) + token * a.ot + h * a.oh;
            } else {
              if (s_k[tok[i]] < 0) continue;
              from = static_cast<const T*>(a.k) + token * a.kt + (h - a.Hq) * a.kh;
              to[i] = static_cast<T*>(a.kc) + s_k[tok[i]] + (h - a.Hq) * a.kch;
            }
            x[i].load(from, u, a.turned, a.pairs);
          }
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (to[i]) {
              x[i].turn(s_cs + tok[i] * a.pairs, u, a.turned);
              x[i].store(to[i], u, a.turned, a.pairs);
            }
        }
  }
  if (a.Hk) {  // values: copied whole
    using Vec = RotaryVec<T, E>;
    const int vu = a.dim / E, vper = max(RO_NT / vu, 1);
    const int row0 = t / vu, first = t - row0 * vu;
    const int rows = n * a.Hk, step = vper * static_cast<int>(gridDim.y);
    if (row0 < vper)
      for (int u = first; u < vu; u += RO_NT)
        for (int r = static_cast<int>(blockIdx.y) * vper + row0; r < rows; r += 4 * step) {
          Vec x[4];
          T* to[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int at = r + i * step;
            to[i] = nullptr;
            if (at >= rows) continue;
            const int tok = at / a.Hk, h = at - tok * a.Hk;
            if (s_v[tok] < 0) continue;
            to[i] = static_cast<T*>(a.vc) + s_v[tok] + h * a.vch + u * E;
            x[i] = *reinterpret_cast<const Vec*>(static_cast<const T*>(a.v) + (token0 + tok) * a.vt + h * a.vh + u * E);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (to[i]) *reinterpret_cast<Vec*>(to[i]) = x[i];
        }
  }
}

template <typename T, int E, bool ADJ>
cudaError_t launch_rotary(RotaryArgs a, cudaStream_t st) {
  // units of a head: two vectors, or one where the neighbours are in it
  const int turned = !ADJ || E == 1 ? a.pairs / E : 2 * a.pairs / E;
  a.turned = turned;
  a.copied = (a.dim - 2 * a.pairs) / E;
  a.per = std::max(RO_NT / (turned + a.copied), 1);
  // Tokens a CTA: one while that leaves SMs without a CTA, up to four (and what its angles have room for).
  const int sms = sm_count();
  const int room = std::max(RO_ANGLES / a.pairs, 1);
  int tokens = 1;
  while (tokens < RO_TOKENS && 2 * tokens <= room && a.T / (2 * tokens) >= 4 * sms) tokens *= 2;
  // shares of the heads while there are fewer CTAs than SMs
  const int rows = tokens * (a.Hq + a.Hk);
  const int64_t ctas = (static_cast<int64_t>(a.T) + tokens - 1) / tokens;
  int64_t shares = std::min<int64_t>((rows + a.per - 1) / a.per, std::max<int64_t>(sms / ctas, 1));
  shares = std::max<int64_t>(std::min<int64_t>(shares, 65535), 1);
  return launch_maybe_pdl(rotary_kernel<T, E, ADJ>, dim3(static_cast<unsigned>(ctas), static_cast<unsigned>(shares)), dim3(RO_NT), 0, st,
                          true, a, tokens);
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
