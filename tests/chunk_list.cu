// The work list of q3s_chunk_attention on the host: every CTA's calls of chunk_walk, with the 32 lanes of its warp as
// contexts that take turns, checked against the definition of the items.
//   chunk_list SEED ROWS ACTIVE MAX_NEW MAX_OWN HEADS GROUP PREFIX WINDOW
// ROWS rows of which every ACTIVE-th (0: the first alone) has tokens.  Prints the segments, batches and cut items, and the
// most lane operations of a CTA; exits with a message where something is wrong.
#include <ucontext.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <random>
#include <vector>

#include "q3s_chunk.cuh"

using namespace q3s;

#define EXPECT(x, ...)                                  \
  do {                                                  \
    if (!(x)) {                                         \
      std::printf("%s:%d: %s: ", __FILE__, __LINE__, #x); \
      std::printf(__VA_ARGS__);                         \
      std::printf("\n");                                \
      std::exit(1);                                     \
    }                                                   \
  } while (0)

struct Warp {
  ucontext_t main, lanes[32];
  std::vector<char> stacks[32];
  long long slot[2][32];
  int turns[32];
  bool done[32];
};
static Warp* g_warp;

// Every operation of the lanes is an exchange of one value of each.
struct HostLanes {
  int lane;
  const long long* exchange(long long x) const {
    Warp& w = *g_warp;
    long long* s = w.slot[w.turns[lane]++ & 1];
    s[lane] = x;
    swapcontext(&w.lanes[lane], &w.main);
    return s;
  }
  template <typename T>
  T shfl(T x, int src) const { return static_cast<T>(exchange(static_cast<long long>(x))[src & 31]); }
  long long scan(long long x) const {
    const long long* s = exchange(x);
    long long r = 0;
    for (int i = 0; i <= lane; ++i) r += s[i];
    return r;
  }
  unsigned ballot(bool x) const {
    const long long* s = exchange(x);
    unsigned r = 0;
    for (int i = 0; i < 32; ++i) r |= static_cast<unsigned>(s[i] != 0) << i;
    return r;
  }
  void sync() const { exchange(0); }
  static int first(unsigned x) { return __builtin_ctz(x); }
  static int count(unsigned x) { return __builtin_popcount(x); }
};

static struct {
  const ChunkArgs* c;
  int cta;
  const ChunkRow* rows;
  ChunkWalk* walker;
  int* segs;
  ChunkSeg* list;
} g_call;
static void lane_main(int lane) {
  chunk_walk(*g_call.c, g_call.cta, g_call.rows, g_call.walker, g_call.segs, g_call.list, HostLanes{lane});
  g_warp->done[lane] = true;
}
// One call by all lanes; returns the operations it took.
static int walk() {
  Warp& w = *g_warp;
  for (int i = 0; i < 32; ++i) {
    w.turns[i] = 0;
    w.done[i] = false;
    w.stacks[i].resize(64 << 10);
    getcontext(&w.lanes[i]);
    w.lanes[i].uc_stack.ss_sp = w.stacks[i].data();
    w.lanes[i].uc_stack.ss_size = w.stacks[i].size();
    w.lanes[i].uc_link = &w.main;
    makecontext(&w.lanes[i], reinterpret_cast<void (*)()>(lane_main), 1, i);
  }
  for (bool more = true; more;) {
    more = false;
    for (int i = 0; i < 32; ++i)
      if (!w.done[i]) {
        swapcontext(&w.main, &w.lanes[i]);
        more = true;
      }
    for (int i = 1; i < 32; ++i) EXPECT(w.turns[i] == w.turns[0] && w.done[i] == w.done[0], "lane %d goes its own way", i);
  }
  return w.turns[0];
}

int main(int argc, char** argv) {
  EXPECT(argc == 10, "arguments");
  int v[9];
  for (int i = 0; i < 9; ++i) v[i] = std::atoi(argv[i + 1]);
  std::mt19937 rng(v[0]);
  auto below = [&](int n) { return static_cast<int>(rng() % static_cast<unsigned>(n)); };
  const int B = v[1], H = v[5], G = v[6], grid = 148;
  std::vector<int32_t> offsets(1, 0), lengths;
  for (int b = 0; b < B; ++b) {
    const int n = (v[2] ? b % v[2] == 0 : b == 0) ? 1 + below(v[3]) : 0;
    offsets.push_back(offsets.back() + n);
    lengths.push_back(n + below(v[4] + 1));
    if (b % 17 == 5) lengths.back() = n / 2;  // fewer than it brings: its first queries see no token of their own
  }
  ChunkArgs c;
  std::memset(&c, 0, sizeof(c));
  c.a.B = B;
  c.a.T = offsets.back();
  c.a.H = H;
  c.a.G = G;
  c.a.L = v[7];
  c.a.bs = 16;
  c.a.max_blocks = 1 << 20;
  c.a.offsets = offsets.data();
  c.a.lengths = lengths.data();
  c.per_tile = CH_M / G;
  c.window = v[8];
  std::vector<ChunkCut> cuts(grid);
  std::memset(cuts.data(), 0x77, cuts.size() * sizeof(ChunkCut));  // a workspace needs no initial value
  c.cuts = cuts.data();

  const int pair = 2 * c.per_tile;
  std::vector<ChunkRow> rows(CH_NT, ChunkRow{0, 0, 0});
  std::vector<long long> cost(B, 0);
  long long all = 0;
  std::map<std::vector<int>, std::vector<char>> want;  // (row, first token, head): its steps, each to be listed once
  for (int b = 0; b < B; ++b) {
    const ChunkRow x = chunk_row(c.a, b);
    if (b < CH_NT) rows[b] = x;
    for (int i0 = 0; i0 < x.n; i0 += pair) {
      cost[b] += chunk_item_cost(c, x, i0) * H;
      const int m = std::min(pair, x.n - i0);
      // by the definition: the steps that hold a key that a query of the item sees
      const long long hi = static_cast<long long>(c.a.L) + std::max(x.len - x.n + i0 + m, 0) - 1;
      const long long lo = c.window ? std::max(static_cast<long long>(c.a.L) + x.len - x.n + i0 - c.window + 1, 0ll) : 0;
      const int before = (c.a.L + CH_KEYS - 1) / CH_KEYS;
      auto step = [&](long long p) { return static_cast<int>(p < c.a.L ? p / CH_KEYS : before + (p - c.a.L) / CH_KEYS); };
      if (hi < 0) continue;
      for (int h = 0; h < H; ++h) want[{b, x.t0 + i0, h}].assign(step(hi) + 1, 0);
      for (int s = 0; s < step(lo); ++s)
        for (int h = 0; h < H; ++h) want[{b, x.t0 + i0, h}][s] = 2;  // before the first
    }
    all += cost[b];
  }
  const int ctas = static_cast<int>(std::min<long long>(grid, std::max(all, 1ll)));
  Warp warp;
  g_warp = &warp;
  struct Part {
    int cta, slot, step0, steps;
  };
  std::map<std::vector<int>, std::vector<Part>> parts;  // of cut items
  long long segments = 0;
  int batches = 0, most = 0;
  std::vector<ChunkSeg> list(CH_SEGS);
  for (int cta = 0; cta < (all > 0 ? ctas : 0); ++cta) {
    const long long range0 = ChunkCutting{all, ctas}.start(cta);
    long long at = 0;
    int b = 0;
    while (at + cost[b] <= range0) at += cost[b++];
    ChunkWalk walker = {b, -1, 0, 0, 1, ctas, at, all};
    int n = 0, ops = 0;
    g_call = {&c, cta, rows.data(), &walker, &n, list.data()};
    while (walker.more) {
      ops += walk();
      ++batches;
      EXPECT(n >= 0 && n <= CH_SEGS, "%d segments", n);
      // what the joining kernel may read, should the CTA give up from here on
      const ChunkCut& k = cuts[cta];
      EXPECT(k.parts == 0 || (k.parts >= 2 && k.cta == cta && cta + k.parts <= ctas && k.slot / 2 == cta && k.h >= 0 && k.h < H && k.token >= 0 &&
                              k.tokens >= 1 && k.tokens <= pair && k.token + k.tokens <= c.a.T),
             "CTA %d of %d, after a call that leaves %s: %d parts from slot %d", cta, ctas, walker.more ? "more" : "none", k.parts, k.slot);
      for (int i = 0; i < n; ++i) {
        const ChunkSeg& g = list[i];
        auto it = want.find({g.b, g.token, g.h});
        EXPECT(it != want.end(), "no such item: row %d, token %d, head %d", g.b, g.token, g.h);
        const ChunkRow x = chunk_row(c.a, g.b);
        EXPECT(g.tokens == std::min(pair, x.n - (g.token - x.t0)) && g.len == x.len && g.i_key == x.len - x.n + g.token - x.t0 + 1, "row %d", g.b);
        EXPECT(g.steps >= 1 && g.step0 >= 0 && g.step0 + g.steps <= static_cast<int>(it->second.size()), "row %d", g.b);
        bool whole = true;
        for (int s = 0; s < static_cast<int>(it->second.size()); ++s) {
          const bool in = s >= g.step0 && s < g.step0 + g.steps;
          EXPECT(!in || it->second[s] == 0, "row %d, head %d: step %d twice or not its own", g.b, g.h, s);
          if (in) it->second[s] = 1; else whole &= it->second[s] == 2;
        }
        EXPECT(whole == (g.slot < 0), "row %d, head %d: slot %d", g.b, g.h, g.slot);
        if (!whole) parts[{g.b, g.token, g.h}].push_back({cta, g.slot, g.step0, g.steps});
      }
      segments += n;
    }
    most = std::max(most, ops);
  }
  for (auto& [item, steps] : want)
    for (char s : steps) EXPECT(s != 0, "row %d, token %d, head %d: a step that nobody has", item[0], item[1], item[2]);
  int joined = 0;
  for (int cta = 0; cta < (all > 0 ? ctas : 0); ++cta) joined += cuts[cta].parts != 0;
  EXPECT(joined == static_cast<int>(parts.size()), "%d cut items, %d to be joined", static_cast<int>(parts.size()), joined);
  for (auto& [item, p] : parts) {
    const ChunkCut& k = cuts[p[0].cta];
    EXPECT(k.parts == static_cast<int>(p.size()) && k.token == item[1] && k.h == item[2], "CTA %d", p[0].cta);
    for (int i = 0; i < k.parts; ++i) EXPECT(p[i].cta == k.cta + i && p[i].slot == (i ? 2 * p[i].cta : k.slot), "CTA %d, part %d", k.cta, i);
  }
  std::printf("%lld %d %d %d\n", segments, batches, joined, most);
  return 0;
}
