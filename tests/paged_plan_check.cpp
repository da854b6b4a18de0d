// The plan of the paged attention's many-row tiles (paged_plan_of, csrc/paged_index.hpp) walked on the host, workgroup by
// workgroup, over seeded calls with bad lengths and cu_seqlens among them: what the join reads has been written, every
// query row's parts cover its keys once, and nothing lies outside the workspace.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <vector>

#include "paged_index.hpp"

using namespace pope;

#define CHECK(x) do { if (!(x)) { std::printf("line %d (%s): %s\n", __LINE__, g_what, #x); std::exit(1); } } while (0)
static char g_what[160] = "";

struct HostWave {
  std::vector<PagedPlanSeg> lanes = std::vector<PagedPlanSeg>(64);
  template <typename F> uint64_t operator()(F&& f) const {
    uint64_t w = 0;
    for (int i = 0; i < 64; ++i) w |= (uint64_t)(f(i) ? 1 : 0) << i;
    return w;
  }
  template <typename F> float sum(F&& f) const {   // in the order of the lanes' exchanges
    float x[64];
    for (int i = 0; i < 64; ++i) x[i] = f(lanes[i]);
    for (int m = 1; m < 64; m *= 2)   // lane 0's; all lanes have the same
      for (int i = 0; i < 64; i += 2 * m) x[i] += x[i + m];
    return x[0];
  }
  template <typename F> bool any(F&& f) const { return std::any_of(lanes.begin(), lanes.end(), f); }
  template <typename F> int of(int i, F&& f) const { return f(lanes.at(i)); }
  template <typename F> int first_above(F&& f, int at, int* before) const {
    int64_t upto = 0;
    for (int i = 0; i < 64; ++i) {
      const int own = f(lanes[i]);
      if (upto + own > at) {
        *before = (int)upto;
        return i;
      }
      upto += own;
    }
    *before = 0;
    return 64;
  }
};

// Returns whether the workgroups were dealt anew.
static bool walk(const PagedSeqs& q, const PagedPlanCall& c, bool ordered) {
  HostWave w;
  if (c.slots)
    for (int i = 0; i < 64; ++i) w.lanes[i] = paged_plan_seg(q, c, i);
  std::map<int, int> parts_of;                       // tile -> parts, as split 0 writes them
  std::map<std::pair<int, int>, PagedRange> ranges;  // (tile, split) -> blocks
  bool dealt = false;
  for (int64_t at = 0; at < c.tiles * c.splits; ++at) {
    const PagedPlan p = paged_plan_of(q, c, (int)at, w);
    dealt = p.dealt;
    const PagedSeg& g = p.t.seg;
    if ((int64_t)p.t.local * c.rows >= (int64_t)g.n * c.G.d) continue;
    CHECK(p.t.local >= 0 && p.tile >= 0 && p.tile < c.tiles && p.split >= 0 && p.least >= 1);
    const int blocks = paged_tile_blocks(g, p.t.local, c.rows, c.G, c.causal);
    CHECK(blocks >= 0 && blocks <= (g.len + kBlockKeys - 1) / kBlockKeys);
    const PagedRange r = paged_range(blocks, c.splits, p.least, 1, p.split);
    if (p.split > 0 && r.begin >= r.end) continue;
    CHECK(p.split < c.splits && r.end <= blocks);
    const int parts = paged_parts(blocks, c.splits, p.least, 1);
    CHECK(parts <= c.splits);
    if (p.split == 0) CHECK(parts_of.emplace(p.tile, parts).second);
    CHECK(ranges.emplace(std::make_pair(p.tile, p.split), r).second);
  }
  for (int tile = 0; tile < c.tiles; ++tile) {   // the join, or one part's own output
    const PagedTile t = paged_tile_of(q, tile, c.G.d, c.rows, 1, w);
    const int64_t count = (int64_t)t.seg.n * c.G.d - (int64_t)t.local * c.rows;
    if (count <= 0) {
      if (ordered) CHECK(!parts_of.count(tile));
      continue;
    }
    CHECK(parts_of.count(tile));
    const int blocks = paged_tile_blocks(t.seg, t.local, c.rows, c.G, c.causal);
    int at = 0;
    for (int s = 0; s < std::max(parts_of[tile], 1); ++s) {
      const auto it = ranges.find({tile, s});
      CHECK(it != ranges.end() && it->second.begin == at);
      at = it->second.end;
    }
    CHECK(at == blocks);
  }
  return dealt;
}

int main(int argc, char**) {
  std::mt19937 rng(11);
  auto pick = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
  int dealt[2] = {0, 0};
  for (int trial = 0; trial < 1500; ++trial) {
    const bool packed = pick(0, 3), mad = pick(0, 2) == 0;
    const int B = pick(0, 5) == 0 ? pick(20, 62) : pick(1, 9), N = packed ? pick(1, 3000) : pick(1, 900), page = 32 << pick(0, 3), cols = pick(1, 40);
    std::vector<int> len(B), cu(B + 1);
    for (int& x : len) x = mad ? pick(-50, 2 * cols * page) : pick(0, 3) ? pick(0, cols * page) : 0;
    for (int& x : cu) x = mad ? (pick(0, 1) ? pick(-100, 2 * N) : pick(0, 1) * N) : pick(0, N);
    if (!mad) std::sort(cu.begin(), cu.end());
    const PagedSeqs q{len.data(), packed ? cu.data() : nullptr, B, N, cols * page};
    PagedPlanCall c;
    c.G = paged_div(pick(1, 8));
    c.rows = 128;
    c.Hk = 1 << pick(0, 4);
    c.tiles = paged_tiles(B, N, packed, c.G.d, c.rows, 1);
    c.splits = pick(1, 40);
    c.least = pick(1, 48);
    c.slots = pick(0, 4) ? pick(8, 512) : 0;
    c.causal = pick(0, 1);
    std::snprintf(g_what, sizeof g_what, "trial %d: packed %d mad %d B %d N %d G %u Hk %d splits %d least %d slots %d", trial, packed, mad, B, N, c.G.d, c.Hk, c.splits, c.least, c.slots);
    dealt[mad] += walk(q, c, !(packed && mad));
  }
  // segments that overlap: their tiles' parts are more than the grid's workgroups
  for (const bool causal : {false, true}) {
    const int cu[] = {0, 1280, 0, 1280, 0, 1280}, len = causal ? 4096 : 1024, lens[] = {len, len, len, len, len};
    const PagedSeqs q{lens, cu, 5, 1280, len};
    PagedPlanCall c;
    c.G = paged_div(1);
    c.rows = 128;
    c.Hk = 1;
    c.tiles = paged_tiles(5, 1280, true, 1, 128, 1);
    c.splits = causal ? 8 : 2;
    c.least = 16;
    c.slots = 512;
    c.causal = causal;
    std::snprintf(g_what, sizeof g_what, "overlapping segments, causal %d", causal);
    CHECK(!walk(q, c, false));
  }
  // Rows behind the last sequence, and sequences of length zero, have tiles and no keys: they leave the others' parts alike.
  // (20 sequences x 2 heads of 4, 60 pages of 32; the grid as the host sizes it: at most two parts for each of 512 places)
  for (const int gap : {0, 3, 150})
    for (const int none : {0, 100})
      for (const bool causal : {false, true}) {
        int cu[21] = {0}, lens[20];
        const int rows[] = {70, 33, none, 5, 300, 0, none, 100, 1, 40, 0, 0, 9, 8, 0, 64, 9, 8, 0, 64}, all[] = {1900, 40, 0, 1200};
        for (int b = 0; b < 20; ++b) {
          cu[b + 1] = cu[b] + rows[b];
          lens[b] = all[b % 4];
        }
        const PagedSeqs q{lens, cu, 20, cu[20] + gap, 1920};
        PagedPlanCall c;
        c.G = paged_div(4);
        c.rows = 128;
        c.Hk = 2;
        c.tiles = paged_tiles(20, q.N, true, 4, 128, 1);
        c.splits = std::min<int>(4, 1024 / (2 * c.tiles));
        c.least = 16;
        c.slots = 512;
        c.causal = causal;
        std::snprintf(g_what, sizeof g_what, "%d rows behind, %d without keys, causal %d", gap, none, causal);
        CHECK(walk(q, c, true));
      }
  // Few rows: a tile's parts by what it sees, whatever the page table's width lets the grid have.
  for (const int splits : {7, 64, 128}) {
    CHECK(paged_parts(63, splits, paged_few_least(63, 8), 4) == (splits == 7 ? 6 : 8));   // 2,000 keys, 8 heads: parts of 8 or 12
    CHECK(paged_parts(16, splits, paged_few_least(16, 8), 4) == 1);                       // 512 keys: one part
    CHECK(paged_parts(500, splits, paged_few_least(500, 8), 4) == (splits == 7 ? 7 : 32));
    CHECK(paged_parts(63, splits, paged_few_least(63, 128), 4) == 4);                     // the chip is full: parts of 16
  }
  for (int blocks = 0; blocks < 2000; ++blocks)
    for (const int64_t tiles : {1, 8, 40, 100, 256, 5000}) {
      const int least = paged_few_least(blocks, tiles);
      CHECK(least >= 8 && least <= 16 && (blocks > 16 || least == 16));
    }
  CHECK(paged_few_least(1 << 26, (1 << 24) - 1) == 16);
  // rows: new token and query head of every row of a tile
  for (int G : {1, 2, 3, 5, 8, 20, 31}) {
    const PagedDiv div = paged_div(G);
    for (int r0 : {0, 16, 128, 1280, 1 << 20})
      for (int x = 0; x < 128; ++x) {
        const PagedRowMap m(r0, div);
        CHECK(m.token(x) == (r0 + x) / G && m.group(x) == (r0 + x) % G);
      }
  }
  std::snprintf(g_what, sizeof g_what, "calls dealt anew: %d good, %d bad bounds", dealt[0], dealt[1]);
  CHECK(dealt[0] > 50);
  if (argc > 1) std::printf("%s\n", g_what);
  std::printf("ok\n");
}
