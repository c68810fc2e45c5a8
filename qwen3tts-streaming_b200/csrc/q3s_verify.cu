// q3s_verify.cu -- drafted tokens verified against the target's probabilities
// (q3s_verify_drafts).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "q3s_args.cuh"
#include "q3s_decode.h"
#include "q3s_device.cuh"
#include "q3s_head.cuh"
#include "q3s_pdl.cuh"
#include "q3s_tma.cuh"

namespace q3s {

namespace cg = cooperative_groups;

struct VerifyArgs {
  int B, T, V;
  int slice;   // entries of the vocabulary that a CTA of a row's cluster takes
  int places;  // places that a CTA looks at together: a power of two, 1..VF_WARPS
  bool held;   // what a draw is made from is held in shared memory (`slice` 64-bit values)
  float temperature_default;
  const void* logits;
  int64_t logits_stride;
  const int64_t* ids;
  const int32_t* offsets;
  const float* uniforms;
  const float* probs;  // or null
  int64_t probs_stride;
  const float* temperature;  // or null
  const int64_t* slot_map;   // or null
  int64_t* tokens_out;
  int32_t* accepted;
  int32_t* rejected;
  int64_t* next_ids;
  int32_t* error_word;
};

constexpr int VF_NT = 512, VF_WARPS = VF_NT / 32;
constexpr int VF_MAX_CLUSTER = 8;
constexpr int VF_SLICE = 8192;  // entries of the vocabulary that a CTA takes, while the cluster grows; it holds so many for the draw
// Relative error that a 32-bit probability may have, besides its distance (in
// log2 units) from the largest one times VF_GAP.  An exponential is off by 2^-22
// (its instruction) and by the rounding of its argument, 2^-24 ln 2 times its
// distance from k; averaged over the distribution that distance is at most its
// entropy and one, so at most 25 (V up to 2^24): 1.0e-6.  c = log2(e) /
// temperature is off by 2^-23, the same for all entries, which counts times the
// distance between the draft's logit and the average one: again at most 24 * 2^-23 ln 2
// = 2.0e-6, or the draft's own distance (VF_GAP).  Sums of eight add 3 * 2^-24, everything
// after them is 64-bit.  In all 3.4e-6, below 2^-18.
constexpr double VF_BOUND = 1.0 / (1 << 18), VF_GAP = 1.0 / (1 << 22);

// Beyond this |x c| its rounding is too coarse for the 32-bit sum to say anything.
constexpr int VF_LARGE = 1 << 20;

// sum_v 2^(x_v c - k) over some entries, k an integer above their largest
// x c (however large that is: no term overflows; VF_NONE: only entries without a
// probability), with the largest logit as a key that orders like it and its
// lowest index.  A NaN among the entries makes the sum one; nothing else does
// where the largest logit is finite.
struct VerifyStat {
  double sum;
  int k;
  uint32_t best;
  int index;
};
constexpr int VF_NONE = -(1 << 30);
Q3S_DEV VerifyStat verify_nothing() { return {0.0, VF_NONE, f2key(-INFINITY), 0x7fffffff}; }

// 2^d for an integer d <= 0 (0 below -1000), exactly.
Q3S_DEV double pow2_int(int d) { return d < -1000 ? 0.0 : __hiloint2double((1023 + d) << 20, 0); }

// All lanes' together, in every lane.
Q3S_DEV VerifyStat verify_join(const VerifyStat& s) {
  VerifyStat r;
  r.k = __reduce_max_sync(FULL, s.k);
  r.best = __reduce_max_sync(FULL, s.best);
  r.index = static_cast<int>(__reduce_min_sync(FULL, s.best == r.best ? static_cast<uint32_t>(s.index) : 0x7fffffffu));
  r.sum = s.sum * pow2_int(s.k - r.k);
#pragma unroll
  for (int d = 16; d; d >>= 1) r.sum += __shfl_xor_sync(FULL, r.sum, d);
  return r;
}
Q3S_DEV VerifyStat verify_shfl(const VerifyStat& s, int lane) {
  return {__shfl_sync(FULL, s.sum, lane), __shfl_sync(FULL, s.k, lane), __shfl_sync(FULL, s.best, lane), __shfl_sync(FULL, s.index, lane)};
}
// Whether the logits have a distribution.
Q3S_DEV bool verify_defined(const VerifyStat& s) { return s.sum == s.sum && fabsf(key2f(s.best)) < INFINITY; }

// 2^(t / 32) for t <= 0 in 64 bits, by a whole warp: with t = 32 n + j + f, j in
// [0, 32) and |f| <= 1/2, 2^n 2^(j/32) e^z, z = f ln 2 / 32, where 2^(j/32) is
// lane j's `root` and e^z its series up to z^5 / 120 (|z| < 0.0109: off by
// z^6 / 720, 2.3e-15).  14 operations in place of exp2's 40 or so.
Q3S_DEV double vf_exp2_64(double t, double root) {
  constexpr double MAGIC = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer, in the low word
  const bool some = t > -32000.0;               // 2^-1000 and less count as 0
  const double shifted = (some ? t : 0.0) + MAGIC;
  const int k = __double2loint(shifted);
  const double z = ((some ? t : 0.0) - (shifted - MAGIC)) * 0.021660849392498290;  // ln 2 / 32
  double p = fma(z, 1.0 / 120, 1.0 / 24);
  p = fma(z, p, 1.0 / 6);
  p = fma(z, p, 0.5);
  p = fma(z, p, 1.0);
  p = fma(z, p, 1.0);
  const double r = __shfl_sync(FULL, root, k & 31) * p;
  return some ? __hiloint2double(__double2hiint(r) + (k >> 5) * (1 << 20), __double2loint(r)) : 0.0;
}
Q3S_DEV float vf_ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// A thread's sums on the way.
struct VerifyRun {
  double sum;
  float k, best;  // k: -infinity before the first entry with a probability
  int index;
};
// N neighbouring entries, the first at index v.
template <int N>
Q3S_DEV void verify_take(VerifyRun& s, const float (&x)[N], int v, float c) {
  float top = x[0];
#pragma unroll
  for (int e = 1; e < N; ++e) top = fmaxf(top, x[e]);
  if (top > s.best) {
    s.best = top;
    int at = N - 1;
#pragma unroll
    for (int e = N - 2; e >= 0; --e) at = x[e] == top ? e : at;
    s.index = v + at;
    const float y = top * c, k = ceilf(fmaf(fabsf(y), 2.384185791015625e-07f, y));  // 2^-22: above the rounding of y
    if (k > s.k) {
      s.sum *= pow2_int(static_cast<int>(fmaxf(s.k - k, -2000.0f)));  // from -infinity times 0: a NaN that came first stays one
      s.k = k;
    }
  }
  const float k = s.k == -INFINITY ? 0.0f : s.k;
  float e[N];
#pragma unroll
  for (int i = 0; i < N; ++i) e[i] = vf_ex2(fmaf(x[i], c, -k));
#pragma unroll
  for (int w = 1; w < N; w *= 2)
#pragma unroll
    for (int i = 0; i + w < N; i += 2 * w) e[i] += e[i + w];
  s.sum += static_cast<double>(e[0]);  // a NaN among the entries stays one
}
Q3S_DEV VerifyStat verify_stat(const VerifyRun& s) {
  // (beyond VF_LARGE k only says that it is)
  return {s.sum, s.k == -INFINITY ? VF_NONE : static_cast<int>(fminf(fmaxf(s.k, -1.0e9f), 1.0e9f)), f2key(s.best), s.index};
}

// A 16-byte vector of logits, as fp32.
template <typename T>
struct VerifyVec;
template <>
struct VerifyVec<float> {
  static constexpr int N = 4;
  Q3S_DEV static void widen(const uint4& f, float (&x)[4]) {
    x[0] = __uint_as_float(f.x), x[1] = __uint_as_float(f.y), x[2] = __uint_as_float(f.z), x[3] = __uint_as_float(f.w);
  }
};
template <>
struct VerifyVec<__nv_bfloat16> {
  static constexpr int N = 8;
  Q3S_DEV static void widen(const uint4& f, float (&x)[8]) {
    const uint32_t w[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
};
template <>
struct VerifyVec<__half> {
  static constexpr int N = 8;
  Q3S_DEV static void widen(const uint4& f, float (&x)[8]) {
    const uint32_t w[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = h.x, x[2 * i + 1] = h.y;
    }
  }
};

// One row's shared state of a CTA.
struct VerifyShared {
  VerifyStat part[VF_MAX_CLUSTER][VF_WARPS];  // [CTA of the cluster][warp], written by that CTA
  VerifyStat place_stat[VF_WARPS];            // of a place
  double sums[2][VF_MAX_CLUSTER * VF_WARPS];  // a pass's sums, CTA by CTA and warp by warp; passes take turns
  VerifyStat stat;                            // of the place that is being decided
  int verdict, place, winner;
  double before, aim;
  int refused;
};

// A cluster a row; its CTAs cut the vocabulary into slices.
//
// First pass, in 32 bits: groups of the CTA's warps take `places` of the row's places at once,
// a running maximum and sum each.  The partial results meet in every CTA's shared memory, and
// every CTA decides for itself, in the same order, which drafts hold; a comparison within the bound of the 32-bit sum's error is
// decided again from a 64-bit sum.  Then the place where the row stops is drawn from: each warp sums its
// neighbouring entries in 64 bits, the sums meet, and the one warp whose entries reach u * total looks for the entry.
//
// Bound by the latency of its passes and, at large vocabularies, by the 64-bit exponentials of the draw: 64 rows of up to 8
// places, 65000 entries, with the draft's probabilities 56 us, of which the bytes are 15 (a cluster of 8 a row, two CTAs a SM,
// in 1.7 turns); 200 rows of up to 6 places, 2051 entries, 11 us; one row of 5 places 9 us.  A CTA that holds its slice's
// exponentials takes them once: the first of these 71 against 94 us at that time.
template <typename T>
__global__ void __launch_bounds__(VF_NT, 2) verify_kernel(const VerifyArgs a) {
  __shared__ VerifyShared sh;
  extern __shared__ double held[];  // [slice], if they are held
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int t = static_cast<int>(threadIdx.x), w = t >> 5, lane = t & 31;
  const int b = static_cast<int>(blockIdx.x) / ctas;
  auto sync = [&]() {
    if (ctas > 1) cluster.sync(); else __syncthreads();
  };
  if (ctas > 1) cluster_arrive_relaxed();  // this CTA has begun: its shared memory may be written (waited for before that)
  grid_wait();
  grid_release();

  // ---- the row's tokens ----
  int t0 = 0, n = 0;
  if (b < a.B) {
    const int o0 = a.offsets[b], o1 = a.offsets[b + 1];
    t0 = min(max(o0, 0), a.T);
    const int end = min(max(o1, t0), a.T);
    n = end - t0;
    if ((t0 != o0 || end != o1) && t == 0 && rank == 0 && a.error_word) atomicOr(a.error_word, Q3S_DECERR_LENGTHS);
  }
  if (t == 0) sh.refused = 0;
  __syncthreads();
  if (rank == 0 && b >= a.B - 1) {  // places past the last row
    const int last = a.B ? t0 + n : 0;
    for (int i = last + t; i < a.T; i += VF_NT) a.tokens_out[i] = -1;
  }
  if (rank == 0 && b == 0 && a.B > 0)  // and before the first
    for (int i = t; i < t0; i += VF_NT) a.tokens_out[i] = -1;
  if (a.slot_map) {
    bool without = false;
    for (int i = t; i < n; i += VF_NT) without |= a.slot_map[t0 + i] < 0;
    if (without) sh.refused = 1;  // every writer writes 1
    __syncthreads();
  }
  if (ctas > 1) cluster_wait();
  if (n == 0 || sh.refused) {  // the same in all CTAs of the cluster
    if (rank == 0) {
      for (int i = t; i < n; i += VF_NT) a.tokens_out[t0 + i] = -1;
      if (t == 0 && b < a.B) {
        a.accepted[b] = 0;
        a.rejected[b] = 0;
        a.next_ids[b] = -1;
      }
    }
    return;
  }
  const double row_uniform = static_cast<double>(a.uniforms[t0]);
  const float heat = a.temperature ? a.temperature[b] : a.temperature_default;
  const bool greedy = !(heat >= 7.888609052210118e-31f);  // 2^-100
  const float c = greedy ? 1.0f : 1.4426950408889634f / heat;
  const double c64 = greedy ? 1.0 : 1.4426950408889634074 / static_cast<double>(heat);
  const int v0 = min(rank * a.slice, a.V), v1 = min(v0 + a.slice, a.V);
  const T* logits = static_cast<const T*>(a.logits);

  // ---- 64-bit passes over one place: each warp's neighbouring entries, 32 at a time ----
  const int share = ((v1 - v0 + VF_WARPS - 1) / VF_WARPS + 31) & ~31;
  const int w0 = min(v0 + w * share, v1), w1 = min(w0 + share, v1);
  const double root = exp2(lane / 32.0), steep = 32.0 * c64;
  // e(v) = 2^((x_v - largest) log2(e) / temperature); a whole warp calls
  auto weight = [&](float x, double best) { return vf_exp2_64((static_cast<double>(x) - best) * steep, root); };
  // the warps' sums meet in every CTA
  int pass = 0;
  auto meet = [&](double s) {
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(FULL, s, d);
    ++pass;  // (the sums of the pass before the last were read before the last one's barrier)
    if (lane < ctas) cluster.map_shared_rank(&sh, lane)->sums[pass & 1][rank * VF_WARPS + w] = s;
    sync();
    double total = 0.0;
    for (int i = lane; i < ctas * VF_WARPS; i += 32) total += sh.sums[pass & 1][i];
#pragma unroll
    for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(FULL, total, d);
    return total;
  };
  // f(v, x_v) of all entries of this warp in turn, x_v requested AHEAD at a time (a float of `from`, -infinity past the end); f is called by the whole warp
  auto each = [&](const auto* from, auto f) {
    constexpr int AHEAD = 4;
    for (int v = w0; v < w1; v += 32 * AHEAD) {
      float x[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) x[i] = v + 32 * i + lane < w1 ? static_cast<float>(from[v + 32 * i + lane]) : -INFINITY;
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (v + 32 * i < w1) f(v + 32 * i + lane, x[i]);
    }
  };

  // ---- which drafts hold ----
  int place = 0;  // where the row stops
  const int group = VF_WARPS / a.places;
  for (int first = 0;; first += a.places) {
    const int mine = first + w / group;
    VerifyRun run = {0.0, -INFINITY, -INFINITY, 0x7fffffff};
    if (mine < n) {
      constexpr int N = VerifyVec<T>::N, AHEAD = 4;
      const T* x = logits + (t0 + mine) * a.logits_stride;
      const int lanes = group * 32, l = (w % group) * 32 + lane;
      // single entries up to the first 16-byte boundary, vectors (several requested at a time), single entries
      const int head = static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(x + v0) & 15)) & 15) / sizeof(T));
      const int vec0 = min(v0 + head, v1), vecs = (v1 - vec0) / N;
      if (l < vec0 - v0) {
        const float one[1] = {static_cast<float>(x[v0 + l])};
        verify_take<1>(run, one, v0 + l, c);
      }
      const uint4* vectors = reinterpret_cast<const uint4*>(x + vec0);
      for (int i = l; i < vecs; i += AHEAD * lanes) {
        uint4 f[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
          if (i + j * lanes < vecs) f[j] = vectors[i + j * lanes];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
          if (i + j * lanes < vecs) {
            float y[N];
            VerifyVec<T>::widen(f[j], y);
            verify_take<N>(run, y, vec0 + (i + j * lanes) * N, c);
          }
      }
      const int rest = vec0 + vecs * N + l;
      if (rest < v1) {
        const float one[1] = {static_cast<float>(x[rest])};
        verify_take<1>(run, one, rest, c);
      }
    }
    // what warp 0 decides with: the draft behind place first + lane
    int64_t draft = -1;
    double aim = 0.0;
    float draft_x = 0.0f;
    if (w == 0 && lane < a.places && first + lane + 1 < n) {
      const int64_t at = t0 + first + lane + 1;
      draft = a.ids[at];
      if (draft >= 0 && draft < a.V) {
        aim = static_cast<double>(a.uniforms[at]) * (a.probs ? static_cast<double>(a.probs[at * a.probs_stride + draft]) : 1.0);
        draft_x = static_cast<float>(logits[(at - 1) * a.logits_stride + draft]);
      }
    }
    const VerifyStat warp_stat = verify_join(verify_stat(run));
    if (first > 0) sync();  // the parts of the turn before have been read
    if (lane < ctas) cluster.map_shared_rank(&sh, lane)->part[rank][w] = warp_stat;
    sync();
    if (w < a.places) {  // a warp joins the parts of a place: of `group` warps of every CTA, up to four a lane
      VerifyStat p = verify_nothing();
      for (int i = 0; i < ctas * group; i += 32) {
        VerifyStat o = verify_nothing();
        if (i + lane < ctas * group) o = sh.part[(i + lane) / group][w * group + (i + lane) % group];
        o = verify_join(o);
        if (lane == i / 32) p = o;
      }
      p = ctas * group > 32 ? verify_join(p) : verify_shfl(p, 0);
      if (lane == 0) sh.place_stat[w] = p;
    }
    __syncthreads();
    int from = 0;  // places of this turn that are decided
    bool stop = false;
    while (!stop) {
      if (w == 0) {
        const int i = first + lane;
        const bool live = lane < a.places && i < n;
        VerifyStat p = verify_nothing();
        int verdict = 1;  // 0: the row stops here, 1: the draft holds, 2: too close
        if (live) {
          p = sh.place_stat[lane];
          verdict = 0;
          if (i + 1 < n && verify_defined(p) && draft >= 0 && draft < a.V) {
            if (greedy) {
              verdict = aim < (draft == p.index ? 1.0 : 0.0);
            } else {
              const double y = static_cast<double>(draft_x) * static_cast<double>(c) - static_cast<double>(p.k);
              const double left = aim * p.sum, right = exp2(y);
              const double error = (VF_BOUND - VF_GAP * fmin(y, 0.0)) * (left + right);
              verdict = !(p.sum > 0.0) || abs(p.k) > VF_LARGE ? 2
                        : !(right > 0.0)                        ? 0
                        : fabs(left - right) <= error           ? 2
                                                                : left < right;
            }
          }
        }
        const unsigned open = __ballot_sync(FULL, live && verdict != 1 && lane >= from);
        const int at = open ? __ffs(open) - 1 : 0;
        if (open && lane == at) {
          sh.place = at;
          sh.verdict = verdict;
          sh.stat = p;
        }
        if (!open && lane == 0) sh.verdict = 1;
      }
      __syncthreads();
      const int verdict = sh.verdict, at = sh.place;
      if (verdict == 1) break;  // all drafts of this turn hold
      place = first + at;
      if (verdict == 0) {
        stop = true;
      } else {
        const T* x = logits + (t0 + place) * a.logits_stride;
        const double best = static_cast<double>(key2f(sh.stat.best));
        double sum = 0.0;
        each(x, [&](int, float y) { sum += weight(y, best); });
        const double total = meet(sum);
        const int64_t d = a.ids[t0 + place + 1];
        const double q = a.probs ? static_cast<double>(a.probs[(t0 + place + 1) * a.probs_stride + d]) : 1.0;
        stop = !(static_cast<double>(a.uniforms[t0 + place + 1]) * q * total < weight(static_cast<float>(x[d]), best));
        from = at + 1;
      }
      __syncthreads();  // before warp 0 writes the next verdict
    }
    if (stop) break;
  }

  // ---- the draw ----
  const VerifyStat stat = sh.stat;
  const bool bad = !verify_defined(stat);
  const T* x = logits + (t0 + place) * a.logits_stride;
  const int64_t draft = place + 1 < n ? a.ids[t0 + place + 1] : -1;
  if (rank == 0) {
    for (int i = t; i < n; i += VF_NT)
      if (i != place) a.tokens_out[t0 + i] = i < place ? a.ids[t0 + i + 1] : -1;
    if (t == 0) {
      a.accepted[b] = place;
      a.rejected[b] = n - 1 - place;
      const bool outside = place + 1 < n && (draft < 0 || draft >= a.V);
      if ((bad || outside) && a.error_word) atomicOr(a.error_word, Q3S_DECERR_VALUES);
    }
  }
  auto finish = [&](int id) {
    a.next_ids[b] = id;
    a.tokens_out[t0 + place] = id;
  };
  if (bad || greedy) {
    if (rank == 0 && t == 0) finish(stat.index == 0x7fffffff ? 0 : stat.index);
    return;
  }
  const double best = static_cast<double>(key2f(stat.best));
  const float* q = a.probs && place + 1 < n ? a.probs + (t0 + place + 1) * a.probs_stride : nullptr;
  const int gone = place + 1 < n && !a.probs && draft >= 0 && draft < a.V ? static_cast<int>(draft) : -1;  // a draft that was certain
  if (q)  // on its way while the weights are taken
    for (int v = w0 + 32 * lane; v < w1; v += 1024) asm volatile("prefetch.global.L2 [%0];" ::"l"(q + v));
  // What is drawn from, `left`: e without the draft; with probabilities e - q times the sum of e, where that is positive.
  // A CTA that holds its slice takes each exponential once.
  double mass = 0.0, sum = 0.0;
  each(x, [&](int v, float y) {
    double e = weight(y, best);  // (every lane: its root goes around)
    if (v == gone) e = 0.0;
    if (a.held && v < w1) held[v - v0] = e;
    sum += e;
  });
  double total = meet(sum);
  bool minus = false;
  if (q) {
    mass = total;
    minus = true;
    sum = 0.0;
    each(q, [&](int v, float y) {
      const double e = a.held ? (v < w1 ? held[v - v0] : 0.0) : weight(v < w1 ? static_cast<float>(x[v]) : -INFINITY, best);
      const double r = fmax(e - (v < w1 ? static_cast<double>(y) : 0.0) * mass, 0.0);
      if (a.held && v < w1) held[v - v0] = r;
      sum += r;
    });
    total = meet(sum);
  }
  const bool again = !(total > 0.0);  // nothing is left: from p
  if (again) {
    minus = false;
    sum = 0.0;
    each(x, [&](int v, float y) {
      const double e = weight(y, best);
      if (a.held && v < w1) held[v - v0] = e;
      sum += e;
    });
    total = meet(sum);
  }
  auto left = [&](int v) {  // a whole warp calls
    if (a.held) return v < w1 ? held[v - v0] : 0.0;
    double e = weight(v < w1 ? static_cast<float>(x[v]) : -INFINITY, best);
    if (v == gone && !again) e = 0.0;
    return minus && v < w1 ? fmax(e - static_cast<double>(q[v]) * mass, 0.0) : e;
  };
  if (w == 0) {  // the warp (of all CTAs') whose entries reach u * total: its number, and the sum before it
    const double aim = row_uniform * total;
    const int warps = ctas * VF_WARPS;
    constexpr int EACH = VF_MAX_CLUSTER * VF_WARPS / 32;  // neighbouring sums of a lane
    double at[EACH], up = 0.0;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      at[j] = lane * EACH + j < warps ? sh.sums[pass & 1][lane * EACH + j] : 0.0;
      up += at[j];
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const double o = __shfl_up_sync(FULL, up, d);
      if (lane >= d) up += o;
    }
    double edge = __shfl_up_sync(FULL, up, 1), mine_before = 0.0;
    if (lane == 0) edge = 0.0;
    int mine = -1, last = -1;  // this lane's first sum that reaches the aim, its last that is not 0
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      if (at[j] > 0.0) {
        last = lane * EACH + j;
        if (mine < 0 && edge + at[j] > aim) mine = last, mine_before = edge;
      }
      edge += at[j];
    }
    const unsigned over = __ballot_sync(FULL, mine >= 0), some = __ballot_sync(FULL, last >= 0);
    const int src = over ? __ffs(over) - 1 : 0;
    const int winner = over ? __shfl_sync(FULL, mine, src) : -1;
    const double before = __shfl_sync(FULL, mine_before, src);
    last = __shfl_sync(FULL, last, some ? 31 - __clz(some) : 0);
    if (lane == 0) {
      sh.winner = winner < 0 ? max(last, 0) : winner;
      sh.before = before;
      sh.aim = winner < 0 ? INFINITY : aim;  // rounding left the aim at or above the sum: the last entry that has any
    }
  }
  __syncthreads();
  if (sh.winner == rank * VF_WARPS + w) {
    double carry = sh.before;
    const double aim = sh.aim;
    int id = -1, last = v0;
    for (int v = w0; v < w1 && id < 0; v += 32) {
      const double s = left(v + lane);
      double up = s;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const double o = __shfl_up_sync(FULL, up, d);
        if (lane >= d) up += o;
      }
      const unsigned over = __ballot_sync(FULL, s > 0.0 && carry + up > aim), some = __ballot_sync(FULL, s > 0.0);
      if (over) id = v + __ffs(over) - 1;
      if (some) last = v + 31 - __clz(some);
      carry += __shfl_sync(FULL, up, 31);
    }
    if (lane == 0) finish(id < 0 ? last : id);
  }
}

template <typename T>
cudaError_t launch_verify(const VerifyArgs& a, int ctas, cudaStream_t st) {
  const int smem = a.held ? a.slice * static_cast<int>(sizeof(double)) : 0;
  static std::atomic<uint64_t> done{0};
  const cudaError_t allowed = allow_smem(verify_kernel<T>, VF_SLICE * static_cast<int>(sizeof(double)), done);
  if (allowed != cudaSuccess) return allowed;
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3(static_cast<unsigned>(std::max(a.B, 1)) * ctas);
  lc.blockDim = dim3(VF_NT);
  lc.dynamicSmemBytes = static_cast<size_t>(smem);
  lc.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = static_cast<unsigned>(ctas);
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  lc.attrs = at;
  lc.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&lc, verify_kernel<T>, a);
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace q3s

extern "C" q3s_status q3s_verify_drafts(const q3s_verify_drafts_desc* d, void* stream) {
  using q3s::report;
  if (!d) return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_verify_drafts: desc is NULL");
  if (d->struct_size != sizeof(q3s_verify_drafts_desc))
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_verify_drafts: struct_size %u != %u (ABI mismatch)", d->struct_size,
                  static_cast<unsigned>(sizeof(q3s_verify_drafts_desc)));
  if (d->batch < 0 || d->batch > Q3S_MAX_CACHE_ROWS || d->tokens < 0)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_verify_drafts: batch %d is not in [0, %d] or tokens %d is negative", d->batch,
                  Q3S_MAX_CACHE_ROWS, d->tokens);
  if (d->vocab < 1 || d->vocab > Q3S_MAX_VERIFY_VOCAB)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_verify_drafts: vocab %d is not in [1, %d]", d->vocab, Q3S_MAX_VERIFY_VOCAB);
  if (d->elem != Q3S_ELEM_F32 && d->elem != Q3S_ELEM_BF16 && d->elem != Q3S_ELEM_F16)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_verify_drafts: unknown elem %d", d->elem);
  if (!d->query_offsets) return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_verify_drafts: query_offsets is required");
  if (d->batch > 0 && (!d->accepted || !d->rejected || !d->next_ids))
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_verify_drafts: accepted, rejected and next_ids are required");
  if (d->tokens > 0 && (!d->logits || !d->ids || !d->uniforms || !d->tokens_out))
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_verify_drafts: logits, ids, uniforms and tokens_out are required");
  if (d->tokens > 1 && (d->logits_row_stride < d->vocab || (d->draft_probs && d->draft_row_stride < d->vocab)))
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_verify_drafts: row strides are below vocab");
  if (d->tokens_out == d->ids && d->ids) return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_verify_drafts: tokens_out must not be ids");
  if (d->batch == 0 && d->tokens == 0) return report(Q3S_OK, "");
  q3s::VerifyArgs a;
  a.B = d->batch;
  a.T = d->tokens;
  a.V = d->vocab;
  a.temperature_default = d->temperature_default;
  a.logits = d->logits;
  a.logits_stride = d->logits_row_stride;
  a.ids = d->ids;
  a.offsets = d->query_offsets;
  a.uniforms = d->uniforms;
  a.probs = d->draft_probs;
  a.probs_stride = d->draft_row_stride;
  a.temperature = d->temperature;
  a.slot_map = d->slot_map;
  a.tokens_out = d->tokens_out;
  a.accepted = d->accepted;
  a.rejected = d->rejected;
  a.next_ids = d->next_ids;
  a.error_word = d->error_word;
  // CTAs of a row: so many that each holds its slice; and more, down to slices of 1024 entries, while
  // all rows' fit the SMs together, two each.  One CTA against eight, 8192 entries: 1 row 19.2 against 9.8 us,
  // 16 rows 17.8 against 10.7, 64 rows 18.2 against 21.9, 200 rows 24.7 against 60.9.
  int ctas = 1;
  while (ctas < q3s::VF_MAX_CLUSTER && static_cast<int64_t>(ctas) * q3s::VF_SLICE < a.V) ctas *= 2;
  while (ctas < q3s::VF_MAX_CLUSTER && ctas * 1024 < a.V && static_cast<int64_t>(a.B) * ctas <= q3s::sm_count()) ctas *= 2;
  a.slice = ((a.V + ctas - 1) / ctas + 31) & ~31;
  a.held = a.slice <= q3s::VF_SLICE;
  // as many places at once as a row of the batch has on average
  const int mean = (a.T + std::max(a.B, 1) - 1) / std::max(a.B, 1);
  a.places = 1;
  while (a.places < std::min(mean, q3s::VF_WARPS)) a.places *= 2;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = d->elem == Q3S_ELEM_F32    ? q3s::launch_verify<float>(a, ctas, st)
                        : d->elem == Q3S_ELEM_BF16 ? q3s::launch_verify<__nv_bfloat16>(a, ctas, st)
                                                   : q3s::launch_verify<__half>(a, ctas, st);
  if (e != cudaSuccess) return report(Q3S_ERR_CUDA, "q3s_verify_drafts: launch failed: %s", cudaGetErrorString(e));
  return report(Q3S_OK, "");
}
