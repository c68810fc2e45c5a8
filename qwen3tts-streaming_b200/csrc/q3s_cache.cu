// q3s_cache.cu -- the paged key/value cache's bookkeeping (q3s_cache_tables,
// q3s_cache_trim) and append (q3s_cache_append).
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "q3s_args.cuh"
#include "q3s_decode.h"
#include "q3s_device.cuh"
#include "q3s_pdl.cuh"

namespace q3s {

struct TablesArgs {
  int B, bs, max_blocks, ring, max_tokens;
  const int32_t* context;
  const int32_t* fresh;  // new tokens per row
  const uint8_t* released;
  int32_t* table;
  int64_t table_stride;
  int32_t* free_blocks;
  const int32_t* free_state;
  int32_t* free_state_out;
  int32_t* lengths_out;
  int32_t* offsets;
  int64_t* slots;
  int32_t* positions;
  int32_t* error_word;
  bool whole_rows;  // rows that end past max_tokens are refused
};

constexpr uint32_t SAT = 0x7fffffffu;
// Sum of two values in [0, 2^31) that stays there: associative, so a scan of
// lengths that add up to more than 31 bits ends at the cap instead of wrapping.
Q3S_DEV uint32_t sat_add(uint32_t a, uint32_t b) { return min(a + b, SAT); }

struct Sums {
  uint32_t tokens, need, back;
};
Q3S_DEV Sums operator+(const Sums& a, const Sums& b) {
  return {sat_add(a.tokens, b.tokens), sat_add(a.need, b.need), sat_add(a.back, b.back)};
}

// One launch, no waiting between CTAs.  Everything a row or a token gets is a
// function of three prefix sums over the rows (new tokens, blocks needed,
// blocks given back), so every CTA scans all rows by itself (9 bytes a row,
// from L2 after the first CTA) and then writes its share: the tokens
// [c * chunk, (c + 1) * chunk), found in the scanned offsets by bisection, and
// the rows r with r % gridDim.x == c.  Inputs that other CTAs still read are
// never written: lengths and ring state have separate outputs, table entries
// that the step writes are at or past the row's held blocks while slots read
// the last held one, and the ring is read at its front and written at its
// back.  A row's own table entries are read (given back) and rewritten
// (readmitted) by the same lane.  Bound by launch and memory latency: two
// dependent loads (lengths, then block ids) and a scan of two barriers for
// each NT * R rows: 3.3 us on the device for 8 rows, 7.0 us for 1500 rows with
// 96000 new tokens (1.3 MB, 0.2 us at HBM's rate).
template <int NT, int R>
__global__ void __launch_bounds__(NT) cache_tables_kernel(const TablesArgs a) {
  constexpr int TILE = NT * R, WARPS = NT / 32;
  __shared__ uint32_t s_off[TILE];    // first token of the row
  __shared__ int32_t s_context[TILE]; // tokens the row already holds
  __shared__ int32_t s_first[TILE];   // rank in the ring of its first fresh block; -1: refused
  __shared__ Sums s_warp[WARPS];
  const int t = static_cast<int>(threadIdx.x), w = t >> 5, lane = t & 31;
  const int cta = static_cast<int>(blockIdx.x), ctas = static_cast<int>(gridDim.x);
  const int chunk = static_cast<int>((static_cast<int64_t>(a.max_tokens) + ctas - 1) / ctas);
  grid_wait();
  grid_release();
  const uint32_t tok0 = static_cast<uint32_t>(min(static_cast<int64_t>(cta) * chunk, static_cast<int64_t>(a.max_tokens)));
  const uint32_t tok1 = min(tok0 + static_cast<uint32_t>(chunk), static_cast<uint32_t>(a.max_tokens));
  const int head = min(max(a.free_state[0], 0), a.ring - 1);
  const int count = min(max(a.free_state[1], 0), a.ring);
  const int bs = a.bs;
  const int64_t room = static_cast<int64_t>(a.max_blocks) * bs;
  int bad = 0;
  uint32_t taken = 0;
  Sums carry = {0, 0, 0};
  auto ring_at = [&](uint32_t rank) {  // ring index `rank` places after the front
    return static_cast<int>((static_cast<uint64_t>(head) + rank) % static_cast<uint32_t>(a.ring));
  };

  for (int row0 = 0; row0 < a.B; row0 += TILE) {
    Sums mine[R], total = {0, 0, 0};
    int context[R], back[R];
    bool fits[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int row = row0 + t * R + i;
      const bool in = row < a.B;
      const int c = in ? a.context[row] : 0, n = in ? a.fresh[row] : 0;
      const bool gone = in && a.released && a.released[row];
      if (c < 0 || n < 0 || c > room) bad |= Q3S_DECERR_LENGTHS;
      const int held_tokens = static_cast<int>(min(static_cast<int64_t>(max(c, 0)), room));
      const uint32_t fresh = static_cast<uint32_t>(max(n, 0));
      context[i] = gone ? 0 : held_tokens;
      back[i] = gone ? static_cast<int>((static_cast<int64_t>(held_tokens) + bs - 1) / bs) : 0;
      const int64_t end = static_cast<int64_t>(context[i]) + fresh;
      fits[i] = end <= room;
      if (!fits[i]) bad |= Q3S_DECERR_TABLE;
      const uint32_t need = fits[i] ? static_cast<uint32_t>((end + bs - 1) / bs - (static_cast<int64_t>(context[i]) + bs - 1) / bs) : 0u;
      mine[i] = {fresh, need, static_cast<uint32_t>(back[i])};
      total = total + mine[i];
    }
    // block-wide exclusive scan of `total`
    Sums up = total;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const Sums o = {__shfl_up_sync(FULL, up.tokens, d), __shfl_up_sync(FULL, up.need, d),
                      __shfl_up_sync(FULL, up.back, d)};
      if (lane >= d) up = up + o;
    }
    if (lane == 31) s_warp[w] = up;
    Sums before = {__shfl_up_sync(FULL, up.tokens, 1), __shfl_up_sync(FULL, up.need, 1),
                   __shfl_up_sync(FULL, up.back, 1)};
    if (lane == 0) before = {0, 0, 0};
    __syncthreads();
    {
      Sums x = lane < WARPS ? s_warp[lane] : Sums{0, 0, 0};
#pragma unroll
      for (int d = 1; d < WARPS; d <<= 1) {
        const Sums o = {__shfl_up_sync(FULL, x.tokens, d), __shfl_up_sync(FULL, x.need, d),
                        __shfl_up_sync(FULL, x.back, d)};
        if (lane >= d) x = x + o;
      }
      const int src = max(w - 1, 0);
      Sums base = {__shfl_sync(FULL, x.tokens, src), __shfl_sync(FULL, x.need, src), __shfl_sync(FULL, x.back, src)};
      if (w == 0) base = {0, 0, 0};
      before = carry + base + before;
      const Sums all = {__shfl_sync(FULL, x.tokens, WARPS - 1), __shfl_sync(FULL, x.need, WARPS - 1),
                        __shfl_sync(FULL, x.back, WARPS - 1)};
      carry = carry + all;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int k = t * R + i, row = row0 + k;
      const Sums at = before;
      before = before + mine[i];
      const uint32_t need = mine[i].need;
      // past the last slot: then so are the tokens of every later row, so the sums of needs that count are those before
      const bool past = a.whole_rows && mine[i].tokens && static_cast<int64_t>(at.tokens) + mine[i].tokens > a.max_tokens;
      const bool granted = fits[i] && !past && (need == 0 || before.need <= static_cast<uint32_t>(count));
      if (!granted && fits[i] && !past) bad |= Q3S_DECERR_POOL;
      if (granted && need) taken = max(taken, before.need);
      s_off[k] = at.tokens;
      s_context[k] = context[i];
      s_first[k] = granted ? static_cast<int>(at.need) : -1;
      // the row's own entries: lane by lane when short, the whole warp when long
      const bool here = row < a.B && row % ctas == cta;
      const int take = granted ? static_cast<int>(need) : 0;
      const int held = (context[i] + bs - 1) / bs;
      if (here) {
        a.lengths_out[row] = granted ? static_cast<int>(context[i] + mine[i].tokens) : context[i];
        a.offsets[row + 1] = static_cast<int>(before.tokens);
        if (row == 0) a.offsets[0] = 0;
        if (take == 1 && back[i] == 0)
          a.table[row * a.table_stride + held] = a.free_blocks[ring_at(at.need)];
      }
      unsigned longer = __ballot_sync(FULL, here && (take > 1 || back[i] > 0));
      while (longer) {
        const int src = __ffs(longer) - 1;
        longer &= longer - 1;
        const int r = __shfl_sync(FULL, row, src), nb = __shfl_sync(FULL, back[i], src);
        const int nt = __shfl_sync(FULL, take, src), h0 = __shfl_sync(FULL, held, src);
        const uint32_t first = __shfl_sync(FULL, at.need, src), behind = __shfl_sync(FULL, at.back, src);
        int32_t* entries = a.table + r * a.table_stride;
        for (int j = lane; j < nb; j += 32) a.free_blocks[ring_at(sat_add(count, behind) + j)] = entries[j];
        // h0 > 0 only when nothing was given back; with h0 == 0 lane j wrote entry j back above
        for (int j = lane; j < nt; j += 32) entries[h0 + j] = a.free_blocks[ring_at(first + j)];
      }
    }
    __syncthreads();  // the tile's rows are in shared memory
    // tokens of this CTA that belong to the tile's rows
    const uint32_t lo = max(tok0, s_off[0]), hi = min(tok1, carry.tokens);
    const int rows = min(TILE, a.B - row0);
    for (uint32_t tok = lo + t; tok < hi; tok += NT) {
      int l = 0, r = rows;  // the last row that starts at or before tok (rows without tokens start where the next one does)
      while (r - l > 1) {
        const int m = (l + r) >> 1;
        if (s_off[m] <= tok) l = m; else r = m;
      }
      const int first = s_first[l], c = s_context[l];
      const int pos = static_cast<int>(min(static_cast<uint32_t>(c) + (tok - s_off[l]), SAT));
      int64_t slot = -1;
      if (first >= 0) {
        const int j = pos / bs, held = (c + bs - 1) / bs;
        const int id = j < held ? a.table[(row0 + l) * a.table_stride + j] : a.free_blocks[ring_at(first + (j - held))];
        slot = static_cast<int64_t>(id) * bs + (pos - j * bs);
      }
      a.slots[tok] = slot;
      a.positions[tok] = pos;
    }
    if (row0 + TILE < a.B) __syncthreads();  // before the next tile's rows replace these
  }
  for (uint32_t tok = max(tok0, carry.tokens) + t; tok < tok1; tok += NT) {  // past the last token
    a.slots[tok] = -1;
    a.positions[tok] = 0;
  }
  if (cta == 0) {
    if (carry.tokens > static_cast<uint32_t>(a.max_tokens)) bad |= Q3S_DECERR_TOKENS;
    __shared__ unsigned s_taken, s_bad;
    if (t == 0) s_taken = 0, s_bad = 0;
    __syncthreads();
    taken = __reduce_max_sync(FULL, taken);
    bad = __reduce_or_sync(FULL, bad);
    if (lane == 0) {
      if (taken) atomicMax(&s_taken, taken);
      if (bad) atomicOr(&s_bad, static_cast<unsigned>(bad));
    }
    __syncthreads();
    if (t == 0) {
      const uint32_t left = static_cast<uint32_t>(count) - s_taken;
      a.free_state_out[0] = ring_at(s_taken);
      a.free_state_out[1] = static_cast<int>(min(sat_add(left, carry.back), static_cast<uint32_t>(a.ring)));
      if (a.B == 0) a.offsets[0] = 0;
      if (a.error_word) *a.error_word = static_cast<int>(s_bad);
    }
  }
}

struct TrimArgs {
  int B, bs, max_blocks, ring;
  const int32_t* lengths;
  const int32_t* removed;
  const int32_t* table;
  int64_t table_stride;
  int32_t* free_blocks;
  const int32_t* free_state;
  int32_t* free_state_out;
  int32_t* lengths_out;
  int32_t* error_word;
};

// Rows cut back.  As above, one launch without a wait between CTAs: where a
// row's blocks go is a prefix sum of the blocks that the rows before it give up,
// so every CTA scans all rows by itself and writes the rows r with
// r % gridDim.x == c.  Nothing that another CTA reads is written (the ring is
// only written, lengths and ring state have separate outputs).  A row's entries
// are copied by its lane where there are up to two, by the warp otherwise.  Bound by launch and latency: 48 rows 2.1 us, 1500 rows 5.8.
template <int NT>
__global__ void __launch_bounds__(NT) cache_trim_kernel(const TrimArgs a) {
  constexpr int WARPS = NT / 32;
  __shared__ uint32_t s_warp[2][WARPS];
  const int t = static_cast<int>(threadIdx.x), w = t >> 5, lane = t & 31;
  const int cta = static_cast<int>(blockIdx.x), ctas = static_cast<int>(gridDim.x);
  grid_wait();
  grid_release();
  const int head = min(max(a.free_state[0], 0), a.ring - 1);
  const int count = min(max(a.free_state[1], 0), a.ring);
  const int64_t room = static_cast<int64_t>(a.max_blocks) * a.bs;
  int bad = 0;
  uint32_t carry = 0;
  for (int row0 = 0, phase = 0; row0 < a.B; row0 += NT, phase ^= 1) {
    const int row = row0 + t;
    const bool in = row < a.B;
    const int length = in ? a.lengths[row] : 0, gone = in ? a.removed[row] : 0;
    const int had = static_cast<int>(min(static_cast<int64_t>(max(length, 0)), room)), cut = min(max(gone, 0), had);
    if (had != length || cut != gone) bad |= Q3S_DECERR_LENGTHS;
    const int kept = had - cut;
    const int first = static_cast<int>((static_cast<int64_t>(kept) + a.bs - 1) / a.bs);
    const int back = static_cast<int>((static_cast<int64_t>(had) + a.bs - 1) / a.bs) - first;
    uint32_t up = static_cast<uint32_t>(back);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t o = __shfl_up_sync(FULL, up, d);
      if (lane >= d) up = sat_add(up, o);
    }
    if (lane == 31) s_warp[phase][w] = up;
    __syncthreads();  // one a tile: the next tile writes the other half
    uint32_t before = __shfl_up_sync(FULL, up, 1);
    if (lane == 0) before = 0;
    {
      uint32_t x = lane < WARPS ? s_warp[phase][lane] : 0u;
#pragma unroll
      for (int d = 1; d < WARPS; d <<= 1) {
        const uint32_t o = __shfl_up_sync(FULL, x, d);
        if (lane >= d) x = sat_add(x, o);
      }
      const uint32_t base = __shfl_sync(FULL, x, max(w - 1, 0));
      before = sat_add(carry, sat_add(w ? base : 0u, before));
      carry = sat_add(carry, __shfl_sync(FULL, x, WARPS - 1));
    }
    const bool here = in && row % ctas == cta;
    if (here) a.lengths_out[row] = kept;
    // entry j of the ring behind its last one, unless it is full
    auto give = [&](uint32_t rank, int32_t id) {
      const uint64_t at = static_cast<uint64_t>(count) + rank;
      if (at < static_cast<uint64_t>(a.ring)) a.free_blocks[(static_cast<uint64_t>(head) + at) % static_cast<uint32_t>(a.ring)] = id;
    };
    if (here && back <= 2)
      for (int j = 0; j < back; ++j) give(sat_add(before, j), a.table[row * a.table_stride + first + j]);
    unsigned longer = __ballot_sync(FULL, here && back > 2);
    while (longer) {
      const int src = __ffs(longer) - 1;
      longer &= longer - 1;
      const int r = __shfl_sync(FULL, row, src), n = __shfl_sync(FULL, back, src), f = __shfl_sync(FULL, first, src);
      const uint32_t behind = __shfl_sync(FULL, before, src);
      const int32_t* entries = a.table + r * a.table_stride + f;
      for (int j = lane; j < n; j += 32) give(sat_add(behind, j), entries[j]);
    }
  }
  if (cta == 0) {
    const int any = __syncthreads_or(bad);
    if (t == 0) {
      const uint64_t held = static_cast<uint64_t>(count) + carry;
      a.free_state_out[0] = head;
      a.free_state_out[1] = static_cast<int>(min(held, static_cast<uint64_t>(a.ring)));
      if (a.error_word) *a.error_word = (any ? Q3S_DECERR_LENGTHS : 0) | (held > static_cast<uint64_t>(a.ring) ? Q3S_DECERR_POOL : 0);
    }
  }
}

struct AppendArgs {
  int T, H, bs, blocks;
  int units;  // units of one head's row: dim / 8 (of 16 bytes) or dim (single elements)
  const void *k, *v;
  int64_t kt, kh, vt, vh;
  const int64_t* slots;
  void *kc, *vc;
  int64_t kb, kch, kp, vb, vch, vp;
  int32_t* error_word;
};

// A copy of 4 * T * H * dim bytes, bound by HBM.  A CTA copies U groups of
// tokens of ONE head's keys or values, a group being as many tokens as its 256
// threads hold rows of `units` units (16 bytes each where every base and stride
// allows it, single elements otherwise): neighbouring tokens mostly share a
// block, so a CTA's stores are one run of memory.  With whole tokens a CTA
// instead (all heads, short runs 16 blocks' strides apart) 12289 tokens of
// 8 x 128 took 25 us against 20.6.  The data and the slots are requested side by
// side.  The heads of the same tokens are neighbours in the grid (22.0
// us for 12289 tokens in shuffled blocks with the tokens there, and three CTAs a
// SM; four 20.0; both 19.3: 5.1 TB/s, where a plain copy's 6.5 TB/s would take
// 15.1); 8 tokens: 1.6 us.
template <typename UNIT, int U>
__global__ void __launch_bounds__(256, 4) cache_append_kernel(const AppendArgs a) {
  using ELEM = typename std::conditional<sizeof(UNIT) == 16, uint16_t, UNIT>::type;
  constexpr int E = sizeof(UNIT) / sizeof(ELEM);
  const int t = static_cast<int>(threadIdx.x), per = max(256 / a.units, 1);  // tokens of a group
  const int row = t / a.units;
  const int64_t token0 = static_cast<int64_t>(blockIdx.y) * per * U + row, limit = static_cast<int64_t>(a.blocks) * a.bs;
  grid_wait();
  grid_release();
  if (row >= per) return;
  for (int part = static_cast<int>(blockIdx.x); part < 2 * a.H; part += static_cast<int>(gridDim.x)) {
    const bool value = part >= a.H;
    const int64_t h = value ? part - a.H : part;
    const ELEM* from = static_cast<const ELEM*>(value ? a.v : a.k) + h * (value ? a.vh : a.kh);
    ELEM* to = static_cast<ELEM*>(value ? a.vc : a.kc) + h * (value ? a.vch : a.kch);
    const int64_t token_stride = value ? a.vt : a.kt, block_stride = value ? a.vb : a.kb, place_stride = value ? a.vp : a.kp;
    for (int u = t - row * a.units; u < a.units; u += 256) {
      UNIT x[U];
      int64_t slot[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int64_t token = token0 + i * per;
        slot[i] = -1;
        if (token < a.T) {
          slot[i] = a.slots[token];
          x[i] = *reinterpret_cast<const UNIT*>(from + token * token_stride + static_cast<int64_t>(u) * E);
        }
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (slot[i] < 0) continue;
        if (slot[i] >= limit) {
          if (a.error_word) atomicOr(a.error_word, Q3S_DECERR_BLOCK_ID);
          continue;
        }
        const int64_t block = (slot[i] >> 32) == 0 ? static_cast<int64_t>(static_cast<uint32_t>(slot[i]) / static_cast<uint32_t>(a.bs))
                                                   : slot[i] / a.bs;
        *reinterpret_cast<UNIT*>(to + block * block_stride + (slot[i] - block * a.bs) * place_stride + static_cast<int64_t>(u) * E) = x[i];
      }
    }
  }
}

template <typename UNIT>
cudaError_t launch_append(const AppendArgs& a, cudaStream_t st) {
  const int per = std::max(256 / a.units, 1);
  const unsigned parts = static_cast<unsigned>(std::min(2 * a.H, 65535));
  auto tiles = [&](int u) { return static_cast<unsigned>((static_cast<int64_t>(a.T) + static_cast<int64_t>(per) * u - 1) / (static_cast<int64_t>(per) * u)); };
  // Four groups a CTA once those CTAs are about one a SM; below, one, for more of
  // them.  One against four, 8 heads of 128: 256 tokens 2.1 against 2.3 us, 512
  // tokens 2.6 against 2.3, 2048 tokens 6.0 against 4.2, 12289 tokens 29 against 16
  // (with the tokens first in the grid).
  if (static_cast<int64_t>(tiles(4)) * parts * 4 < 3 * sm_count())
    return launch_maybe_pdl(cache_append_kernel<UNIT, 1>, dim3(parts, tiles(1)), dim3(256), 0, st, true, a);
  // a grid has 65535 rows of CTAs: millions of tokens take several
  const int64_t most = static_cast<int64_t>(65535) * per * 4;
  cudaError_t e = cudaSuccess;
  for (int64_t t0 = 0; t0 < a.T && e == cudaSuccess; t0 += most) {
    AppendArgs b = a;
    constexpr int64_t size = sizeof(uint16_t);  // of an element, as the strides count them
    b.T = static_cast<int>(std::min(most, a.T - t0));
    b.k = static_cast<const unsigned char*>(a.k) + t0 * a.kt * size;
    b.v = static_cast<const unsigned char*>(a.v) + t0 * a.vt * size;
    b.slots = a.slots + t0;
    e = launch_maybe_pdl(cache_append_kernel<UNIT, 4>, dim3(parts, static_cast<unsigned>((b.T + per * 4 - 1) / (per * 4))), dim3(256), 0,
                         st, true, b);
  }
  return e;
}

}  // namespace q3s

extern "C" q3s_status q3s_cache_tables(const q3s_cache_tables_desc* d, void* stream) {
  using q3s::report;
  if (!d) return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_cache_tables: desc is NULL");
  if (d->struct_size != sizeof(q3s_cache_tables_desc) && d->struct_size != offsetof(q3s_cache_tables_desc, flags))
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_cache_tables: struct_size %u != %u (ABI mismatch)", d->struct_size,
                  static_cast<unsigned>(sizeof(q3s_cache_tables_desc)));
  const uint32_t flags = d->struct_size == sizeof(q3s_cache_tables_desc) ? d->flags : 0u;
  if (flags & ~Q3S_TABLES_WHOLE_ROWS) return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_cache_tables: unknown flags %#x", flags);
  if (d->batch < 0 || d->batch > Q3S_MAX_CACHE_ROWS)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_cache_tables: batch %d is not in [0, %d]", d->batch, Q3S_MAX_CACHE_ROWS);
  if (d->block_size < 1 || d->max_blocks < 1 || d->ring_size < 1 || d->max_tokens < 0)
    return report(Q3S_ERR_INVALID_ARGUMENT,
                  "q3s_cache_tables: block_size, max_blocks and ring_size must be positive and max_tokens not negative");
  if (static_cast<int64_t>(d->max_blocks) * d->block_size > 0x7fffffffll)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_cache_tables: a table of %d blocks of %d tokens passes 31 bits",
                  d->max_blocks, d->block_size);
  if (!d->free_blocks || !d->free_state || !d->free_state_out || !d->query_offsets)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_cache_tables: free_blocks, free_state, free_state_out and query_offsets are required");
  if (d->batch > 0 && (!d->context_lengths || !d->new_lengths || !d->block_table || !d->lengths_out))
    return report(Q3S_ERR_INVALID_ARGUMENT,
                  "q3s_cache_tables: context_lengths, new_lengths, block_table and lengths_out are required");
  if (d->max_tokens > 0 && (!d->slot_map || !d->positions))
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_cache_tables: slot_map and positions are required");
  if (d->batch > 1 && d->block_table_stride < d->max_blocks)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_cache_tables: block_table_stride is below max_blocks");
  if (d->lengths_out && (d->lengths_out == d->context_lengths || d->lengths_out == d->new_lengths))
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_cache_tables: lengths_out must not be an input");
  if (d->free_state_out == d->free_state)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_cache_tables: free_state_out must not be free_state");
  q3s::TablesArgs a;
  a.B = d->batch;
  a.bs = d->block_size;
  a.max_blocks = d->max_blocks;
  a.ring = d->ring_size;
  a.max_tokens = d->max_tokens;
  a.context = d->context_lengths;
  a.fresh = d->new_lengths;
  a.released = d->released;
  a.table = d->block_table;
  a.table_stride = d->block_table_stride;
  a.free_blocks = d->free_blocks;
  a.free_state = d->free_state;
  a.free_state_out = d->free_state_out;
  a.lengths_out = d->lengths_out;
  a.offsets = d->query_offsets;
  a.slots = d->slot_map;
  a.positions = d->positions;
  a.error_word = d->error_word;
  a.whole_rows = (flags & Q3S_TABLES_WHOLE_ROWS) != 0;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  // CTAs: one per NT tokens or per 32 rows (their entries), up to one per SM.
  // Threads and rows a thread, so that the rows are one scan.  Small against
  // large: 8 rows 3.0 against 4.4 us, 128 rows 3.4 against 4.8, 256 rows 4.4
  // against 4.9, 512 rows 6.6 against 5.0; one row a thread against two: 1000
  // rows 5.1 against 5.8 us, 1500 rows 7.3 against 5.8.
  const int sms = q3s::sm_count();
  auto ctas = [&](int nt) {
    return std::max(1, std::min(sms, std::max(static_cast<int>((static_cast<int64_t>(a.max_tokens) + nt - 1) / nt), (a.B + 31) / 32)));
  };
  const cudaError_t e =
      a.B <= 256 && a.max_tokens <= 1024
          ? q3s::launch_maybe_pdl(q3s::cache_tables_kernel<128, 1>, dim3(ctas(128)), dim3(128), 0, st, true, a)
      : a.B <= 1024 ? q3s::launch_maybe_pdl(q3s::cache_tables_kernel<1024, 1>, dim3(ctas(1024)), dim3(1024), 0, st, true, a)
                    : q3s::launch_maybe_pdl(q3s::cache_tables_kernel<1024, 2>, dim3(ctas(1024)), dim3(1024), 0, st, true, a);
  if (e != cudaSuccess) return report(Q3S_ERR_CUDA, "q3s_cache_tables: launch failed: %s", cudaGetErrorString(e));
  return report(Q3S_OK, "");
}

extern "C" q3s_status q3s_cache_trim(const q3s_cache_trim_desc* d, void* stream) {
  using q3s::report;
  if (!d) return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_cache_trim: desc is NULL");
  if (d->struct_size != sizeof(q3s_cache_trim_desc))
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_cache_trim: struct_size %u != %u (ABI mismatch)", d->struct_size,
                  static_cast<unsigned>(sizeof(q3s_cache_trim_desc)));
  if (d->batch < 0 || d->batch > Q3S_MAX_CACHE_ROWS)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_cache_trim: batch %d is not in [0, %d]", d->batch, Q3S_MAX_CACHE_ROWS);
  if (d->block_size < 1 || d->max_blocks < 1 || d->ring_size < 1)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_cache_trim: block_size, max_blocks and ring_size must be positive");
  if (static_cast<int64_t>(d->max_blocks) * d->block_size > 0x7fffffffll)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_cache_trim: a table of %d blocks of %d tokens passes 31 bits", d->max_blocks,
                  d->block_size);
  if (!d->free_blocks || !d->free_state || !d->free_state_out)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_cache_trim: free_blocks, free_state and free_state_out are required");
  if (d->batch > 0 && (!d->lengths || !d->removed || !d->block_table || !d->lengths_out))
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_cache_trim: lengths, removed, block_table and lengths_out are required");
  if (d->batch > 1 && d->block_table_stride < d->max_blocks)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_cache_trim: block_table_stride is below max_blocks");
  if (d->lengths_out && (d->lengths_out == d->lengths || d->lengths_out == d->removed))
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_cache_trim: lengths_out must not be an input");
  if (d->free_state_out == d->free_state)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_cache_trim: free_state_out must not be free_state");
  q3s::TrimArgs a;
  a.B = d->batch;
  a.bs = d->block_size;
  a.max_blocks = d->max_blocks;
  a.ring = d->ring_size;
  a.lengths = d->lengths;
  a.removed = d->removed;
  a.table = d->block_table;
  a.table_stride = d->block_table_stride;
  a.free_blocks = d->free_blocks;
  a.free_state = d->free_state;
  a.free_state_out = d->free_state_out;
  a.lengths_out = d->lengths_out;
  a.error_word = d->error_word;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const unsigned ctas = static_cast<unsigned>(std::max(1, std::min(q3s::sm_count(), (a.B + 31) / 32)));
  const cudaError_t e = a.B <= 128 ? q3s::launch_maybe_pdl(q3s::cache_trim_kernel<128>, dim3(ctas), dim3(128), 0, st, true, a)
                                   : q3s::launch_maybe_pdl(q3s::cache_trim_kernel<1024>, dim3(ctas), dim3(1024), 0, st, true, a);
  if (e != cudaSuccess) return report(Q3S_ERR_CUDA, "q3s_cache_trim: launch failed: %s", cudaGetErrorString(e));
  return report(Q3S_OK, "");
}

extern "C" q3s_status q3s_cache_append(const q3s_cache_append_desc* d, void* stream) {
  using q3s::report;
  if (!d) return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_cache_append: desc is NULL");
  if (d->struct_size != sizeof(q3s_cache_append_desc))
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_cache_append: struct_size %u != %u (ABI mismatch)", d->struct_size,
                  static_cast<unsigned>(sizeof(q3s_cache_append_desc)));
  if (d->tokens < 0 || d->kv_heads < 1 || d->dim < 1 || d->block_size < 1 || d->blocks < 1)
    return report(Q3S_ERR_INVALID_ARGUMENT,
                  "q3s_cache_append: kv_heads, dim, block_size and blocks must be positive and tokens not negative");
  if (static_cast<int64_t>(d->kv_heads) * d->dim > (1 << 24))
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_cache_append: kv_heads * dim is above 2^24");
  if (d->elem != Q3S_ELEM_F32 && d->elem != Q3S_ELEM_BF16 && d->elem != Q3S_ELEM_F16)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_cache_append: unknown elem %d", d->elem);
  if (d->tokens == 0) return report(Q3S_OK, "");
  if (!d->k || !d->v || !d->slot_map || !d->k_cache || !d->v_cache)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_cache_append: k, v, slot_map, k_cache and v_cache are required");
  q3s::AppendArgs a;
  a.T = d->tokens;
  a.H = d->kv_heads;
  a.bs = d->block_size;
  a.blocks = d->blocks;
  a.k = d->k;
  a.v = d->v;
  a.slots = d->slot_map;
  a.kc = d->k_cache;
  a.vc = d->v_cache;
  a.error_word = d->error_word;
  // 32-bit elements are copied as pairs of 16-bit ones
  const int64_t wide = d->elem == Q3S_ELEM_F32 ? 2 : 1;
  const int64_t strides[10] = {d->k_token_stride, d->k_head_stride,       d->v_token_stride, d->v_head_stride,
                               d->k_block_stride, d->k_cache_head_stride, d->k_place_stride, d->v_block_stride,
                               d->v_cache_head_stride, d->v_place_stride};
  int64_t* to[10] = {&a.kt, &a.kh, &a.vt, &a.vh, &a.kb, &a.kch, &a.kp, &a.vb, &a.vch, &a.vp};
  const int64_t dim = d->dim * wide;
  bool vec = dim % 8 == 0;
  for (int i = 0; i < 10; ++i) {
    *to[i] = strides[i] * wide;
    vec = vec && *to[i] % 8 == 0;
  }
  for (const void* p : {d->k, d->v, static_cast<const void*>(d->k_cache), static_cast<const void*>(d->v_cache)})
    vec = vec && (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
  const int units = static_cast<int>(vec ? dim / 8 : dim);
  a.units = units;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = vec ? q3s::launch_append<uint4>(a, st) : q3s::launch_append<uint16_t>(a, st);
  if (e != cudaSuccess) return report(Q3S_ERR_CUDA, "q3s_cache_append: launch failed: %s", cudaGetErrorString(e));
  return report(Q3S_OK, "");
}

extern "C" uint32_t q3s_decode_desc_size(int32_t which) {
  switch (which) {
    case 0: return sizeof(q3s_cache_tables_desc);
    case 1: return sizeof(q3s_cache_append_desc);
    case 2: return sizeof(q3s_prefix_attention_desc);
    case 3: return sizeof(q3s_quantize_rows_desc);
    case 4: return sizeof(q3s_int8_matmul_desc);
    case 5: return sizeof(q3s_rotary_desc);
    case 6: return sizeof(q3s_verify_drafts_desc);
    case 7: return sizeof(q3s_cache_trim_desc);
    case 8: return sizeof(q3s_chunk_attention_desc);
  }
  return 0;
}
