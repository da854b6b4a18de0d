// The index arithmetic of the paged cache (csrc/paged_index.hpp) walked on the host as the kernels walk it, over
// seeded calls with bad lengths and cu_seqlens among them: every row belongs to one tile, nothing lies out of range,
// every key is in one split, and the operand-order layouts are permutations of a block.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "paged_index.hpp"

using namespace pope;

#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); std::exit(1); } } while (0)

// paged_tile of the kernels: the last segment whose first tile is at or below `tile`
static bool find_tile(const PagedSeqs& q, int64_t tile, int unit, int per, int extra, PagedSeg* g, int64_t* local) {
  if (!q.cu) {
    *local = tile / q.B;   // the sequences' n-th tiles side by side
    *g = paged_seg(q, (int)(tile - *local * q.B));
    return true;
  }
  int found = 0;
  for (int s0 = 0; s0 < q.B + 2; s0 += 64) {   // as the lanes do: the last hit of the last chunk that has one
    int last = -1;
    for (int s = s0; s < s0 + 64 && s < q.B + 2; ++s)
      if (paged_first_tile(q, s, unit, per, extra) <= tile) last = s;
    if (last < 0) break;
    found = last;
    if (found != s0 + 63) break;
  }
  *g = paged_seg(q, found);
  *local = tile - paged_first_tile(q, found, unit, per, extra);
  return true;
}

int main() {
  std::mt19937 rng(7);
  auto pick = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
  for (int trial = 0; trial < 4000; ++trial) {
    const bool packed = pick(0, 1), mad = pick(0, 3) == 0;
    const int B = pick(0, 9) == 0 ? pick(60, 140) : pick(1, 9), N = packed ? pick(1, 400) : pick(1, 150), page = 32 << pick(0, 3), cols = pick(1, 6);
    std::vector<int> len(B), cu(B + 1);
    for (int& x : len) x = mad ? pick(-50, 2 * cols * page) : pick(0, cols * page);
    if (mad && pick(0, 1)) len[0] = pick(0, 1) ? 2147483647 : -2147483647 - 1;
    for (int& x : cu) x = mad ? pick(-100, 2 * N) : pick(0, N);
    const bool ordered = !mad;
    if (ordered) std::sort(cu.begin(), cu.end());
    PagedSeqs q{len.data(), packed ? cu.data() : nullptr, B, N, cols * page};
    const int batches = packed ? 1 : B;

    // attention: row tiles
    const int G = pick(1, 8), rows = 16 << pick(0, 3), Hk = 1;
    (void)Hk;
    std::vector<int> seen((size_t)batches * N * G, 0);
    const int64_t tiles = paged_tiles(B, N, packed, G, rows, 1);
    for (int64_t t = 0; t < tiles; ++t) {
      PagedSeg g;
      int64_t local;
      find_tile(q, t, G, rows, 1, &g, &local);
      CHECK(g.b >= -1 && g.b < B && g.batch >= 0 && g.batch < batches && g.n >= 0 && g.row0 >= 0 && g.row0 + g.n <= N);
      CHECK(g.len >= 0 && g.len <= q.capacity && (g.b >= 0 || g.len == 0));
      CHECK(local >= 0 || !ordered);
      if (local < 0) local = 0;
      for (int64_t r = local * rows; r < std::min<int64_t>((local + 1) * rows, (int64_t)g.n * G); ++r) {
        ++seen[((size_t)g.batch * N + g.row0 + r / G) * G + r % G];
        for (bool causal : {false, true}) {
          const int lim = paged_limit(g.first + (int)(r / G), g.len, causal);
          CHECK(lim >= 0 && lim <= g.len);
          if (causal && g.first + r / G >= 0) CHECK(lim == g.first + r / G + 1);
        }
      }
    }
    if (ordered) for (int x : seen) CHECK(x == 1);

    // write / read: blocks of 32 slots
    std::vector<int> got((size_t)batches * N, 0);
    const int64_t blocks = paged_tiles(B, N, packed, 1, kBlockKeys, 2);
    for (int64_t t = 0; t < blocks; ++t) {
      PagedSeg g;
      int64_t local;
      find_tile(q, t, 1, kBlockKeys, 2, &g, &local);
      const int blk = floor_div(g.first, kBlockKeys) + (int)local, i0 = blk * kBlockKeys - g.first;
      if (i0 >= g.n) continue;
      CHECK(local >= 0 || !ordered);
      for (int s = 0; s < kBlockKeys; ++s) {
        if ((unsigned)(i0 + s) >= (unsigned)g.n) continue;
        ++got[(size_t)g.batch * N + g.row0 + i0 + s];
        const int pos = blk * kBlockKeys + s;
        CHECK(pos == g.first + i0 + s);
        if (blk >= 0 && g.b >= 0) CHECK(pos < q.capacity && blk / (page / kBlockKeys) < cols);
        if (g.b < 0) CHECK(blk < 0);
      }
    }
    if (ordered) for (int x : got) CHECK(x == 1);

    // splits
    const int nb = pick(0, 700), splits = pick(1, 70), least = pick(1, 20), step = 1 << pick(0, 2);
    std::vector<int> part(nb, 0);
    const int per = paged_split_blocks(nb, splits, least, step);
    CHECK(per >= least && per % step == 0);
    for (int s = 0; s < splits; ++s) {
      const PagedRange r = paged_range(nb, splits, least, step, s);
      CHECK(r.begin >= 0 && r.begin <= r.end && r.end <= nb);
      CHECK((r.begin < r.end) == (s < paged_parts(nb, splits, least, step)));   // the join counts the same splits
      for (int b = r.begin; b < r.end; ++b) ++part[b];
    }
    for (int x : part) CHECK(x == 1);
  }
  for (uint32_t d : {1u, 2u, 3u, 5u, 7u, 8u, 20u, 31u, 127u, 1000u, 65535u, 65537u, 1u << 30}) {
    const PagedDiv div = paged_div(d);
    for (int k = 0; k < 20000; ++k) {
      const uint32_t x = k < 200 ? k : k < 400 ? 0x7fffffffu - (k - 200) : (rng() & 0x7fffffffu) / d * d + (k & 1 ? d - 1 : 0);
      if (x <= 0x7fffffffu) CHECK(div.of(x) == x / d);
    }
  }
  for (bool q8 : {false, true}) {
    for (int steps = 1; steps <= 16; ++steps) {
      std::vector<int> hit(kBlockKeys * steps * 32, 0);
      for (int t = 0; t < kBlockKeys; ++t)
        for (int e = 0; e < steps * 32; ++e) ++hit.at(paged_k_off(q8, t, e));
      for (int x : hit) CHECK(x == 1);
    }
    for (int tiles = 2; tiles <= 16; tiles += 2) {
      std::vector<int> hit(kBlockKeys * tiles * 16, 0);
      for (int t = 0; t < kBlockKeys; ++t)
        for (int d = 0; d < tiles * 16; ++d) ++hit.at(paged_v_off(q8, t, d));
      for (int x : hit) CHECK(x == 1);
    }
  }
  std::vector<int> hit(64, 0);
  for (int t = 0; t < kBlockKeys; ++t)
    for (int w = 0; w < 2; ++w) ++hit.at(paged_scale_off(t, w));
  for (int x : hit) CHECK(x == 1);
  for (int D = 1; D <= 256; ++D)
    for (int R = 0; R <= D; ++R) {
      const int s = paged_k_steps(D, R), v = paged_v_tiles(D);
      CHECK(s * 32 >= D + R && v * 16 >= D && s <= v && s >= v / 2);   // s <= v: a key row fits 2 D columns of LDS
    }
  std::printf("ok\n");
}
