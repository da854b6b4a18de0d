// Index arithmetic of the paged cache: which rows a workgroup has, which keys a row sees, where a slot's
// elements lie.  Integers only, no HIP: the kernels and the host tests compile the same functions.
//
// Segments.  A call's new rows are a padded batch (sequence b: rows 0 .. N - 1 of batch b), or packed: T rows
// that cu_seqlens[0 .. B] cuts into sequences.  Packed rows outside every sequence form two more segments
// without a cache (before cu[0] and from cu[B] on), so every row belongs to exactly one of B + 2 segments
// whose bounds are cu clipped to [0, T].  Row i of the n rows of a sequence of length L stands at position
// L - n + i; rows at negative positions have no slot.
//
// Tiles of packed calls.  The host does not know the sequences' lengths.  A segment that starts at unit c gets
// the tiles floor(c / per) + extra * s .. : consecutive starts differ by at least floor(n / per) + extra, which
// covers every tile of n units (extra = 1 for aligned tiles; 2 where the first tile may be cut by an alignment in the
// cache, as the blocks of 32 slots are).
#pragma once
#include <stdint.h>

#if defined(__HIPCC__)
#define POPE_HD __host__ __device__ __forceinline__
#else
#define POPE_HD inline
#endif

namespace pope {

constexpr int kBlockKeys = 32;   // keys per block: the k extent of one 16-bit MFMA of the P V product

POPE_HD int clip(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }
POPE_HD int floor_div(int a, int b) { return a >= 0 ? a / b : -((b - 1 - a) / b); }

// Division of numbers below 2^31 by d in [1, 2^30]: a product and a shift (with s = ceil(log2 d), m = ceil(2^(31 + s) / d) is too
// large by less than d / d <= 1, which moves x m / 2^(31 + s) by less than 2^31 / 2^(31 + s) <= 1 / d).
struct PagedDiv {
  uint32_t d, m;
  int shift;
  POPE_HD uint32_t of(uint32_t x) const { return (uint32_t)(((uint64_t)x * m) >> shift); }
};
inline PagedDiv paged_div(uint32_t d) {
  int s = 0;
  while (((uint32_t)1 << s) < d) ++s;
  return PagedDiv{d, (uint32_t)((((uint64_t)1 << (31 + s)) + d - 1) / d), 31 + s};
}

// What a call says about its sequences.
struct PagedSeqs {
  const int* lengths;   // (B)
  const int* cu;        // (B + 1), or null: a padded batch
  int B, N;             // N: rows per sequence, or rows in all (packed)
  int capacity;         // slots a page table row covers
};

// A run of rows of one sequence: rows row0 .. row0 + n - 1 at positions first .. first + n - 1 < len.
struct PagedSeg {
  int b;                // sequence whose page table row holds, or -1: no cache
  int batch;            // batch index of the rows' tensors
  int row0, n;
  int len;              // cached slots
  int first;            // position of the first row (may be negative)
};

POPE_HD int paged_bound(const PagedSeqs& q, int s) {   // first packed row of segment s, 0 <= s <= B + 2
  return s == 0 ? 0 : s > q.B + 1 ? q.N : clip(q.cu[s - 1], 0, q.N);
}
// First tile of packed segment s; `unit` units per row (query heads of a key head), `per` units per tile.
POPE_HD int64_t paged_first_tile(const PagedSeqs& q, int s, int unit, int per, int extra) {
  return (int64_t)paged_bound(q, s) * unit / per + (int64_t)extra * s;
}
POPE_HD int64_t paged_tiles(int B, int N, bool packed, int unit, int per, int extra) {
  return packed ? (int64_t)N * unit / per + (int64_t)extra * (B + 2)
                : (int64_t)B * (((int64_t)N * unit + per - 1) / per + extra - 1);
}
POPE_HD PagedSeg paged_seg(const PagedSeqs& q, int s) {   // packed segment s < B + 2, or padded sequence s < B
  PagedSeg g;
  if (q.cu) {
    const int lo = paged_bound(q, s), hi = paged_bound(q, s + 1);
    g.b = s >= 1 && s <= q.B ? s - 1 : -1;
    g.batch = 0;
    g.row0 = lo;
    g.n = hi > lo ? hi - lo : 0;
  } else {
    g.b = g.batch = s;
    g.row0 = 0;
    g.n = q.N;
  }
  g.len = g.b >= 0 ? clip(q.lengths[g.b], 0, q.capacity) : 0;
  g.first = g.len - g.n;
  return g;
}

// The segment that tile `tile` belongs to, and its tile within it; seg.n = 0 where there is none.  Packed calls: 64 segments'
// first tiles are tested at a time (`hits(f)`: bit i set where f(i) holds, a wave's ballot), and the last one at or below
// `tile` has it (with bounds that decrease, any segment may come out, and paged_seg bounds it).  Padded calls: the
// sequences' n-th tiles side by side.
struct PagedTile { PagedSeg seg; int local; };
template <typename Hits>
POPE_HD PagedTile paged_tile_of(const PagedSeqs& q, int tile, int unit, int per, int extra, Hits&& hits) {
  PagedTile t;
  if (!q.cu) {
    t.local = (int)((unsigned)tile / (unsigned)q.B);
    t.seg = paged_seg(q, tile - t.local * q.B);
    return t;
  }
  const int S = q.B + 2;
  int found = 0;
  for (int s0 = 0; s0 < S; s0 += 64) {
    const uint64_t w = hits([&](int i) { return s0 + i < S && paged_first_tile(q, s0 + i < S ? s0 + i : 0, unit, per, extra) <= tile; });
    if (!w) break;
    found = s0 + 63 - __builtin_clzll(w);
    if (found != s0 + 63) break;
  }
  t.seg = paged_seg(q, found);
  t.local = (int)(tile - paged_first_tile(q, found, unit, per, extra));
  return t;
}

// Keys a row at position pos sees: [0, limit).
POPE_HD int paged_limit(int pos, int len, bool causal) { return !causal ? len : pos < 0 ? 0 : pos + 1 < len ? pos + 1 : len; }

// Key blocks of split s of `splits`: every split but the last has `per` of them.
struct PagedRange { int begin, end; };
POPE_HD int paged_split_blocks(int blocks, int splits, int least, int step) {
  int per = (blocks + splits - 1) / splits;
  per = per < least ? least : per;
  return (per + step - 1) / step * step;
}
POPE_HD int paged_parts(int blocks, int splits, int least, int step) {   // splits that have blocks; 0: there are none
  const int per = paged_split_blocks(blocks, splits, least, step);
  return (blocks + per - 1) / per;
}
POPE_HD PagedRange paged_range(int blocks, int splits, int least, int step, int s) {
  const int per = paged_split_blocks(blocks, splits, least, step);
  const int64_t lo = (int64_t)s * per, hi = lo + per;
  return PagedRange{lo < blocks ? (int)lo : blocks, hi < blocks ? (int)hi : blocks};
}

// Least blocks of a part, few rows, of a tile of `blocks` blocks in a launch of `tiles` tiles over all heads: 16, or as few as 8
// where 16 leave some of the 256 CUs without a part (the rule's figures are beside the host's, pope_abi.cpp).  By what the
// tile sees, not by the page table's width, which a serving program sizes for its longest context.
POPE_HD int paged_few_least(int blocks, int64_t tiles) {
  if (blocks <= 16) return 16;
  const int64_t even = tiles * blocks / 256;
  return even < 8 ? 8 : even > 16 ? 16 : (int)even;
}

// A workgroup's tile and part of the key axis, where a tile has many rows.
//
// At most 64 segments (`slots`, the workgroups that the chip holds, is not 0): parts are cut by what the sequences
// have, as few blocks as these workgroups get of all tiles' blocks, or more where the tiles' parts would then be more
// than the workgroups.  A quarter of what causality takes from a prompt's first rows is left out: its heaviest tile has
// twice the mean's blocks and would end alone (prompts of 4,096 tokens x 8 heads, D 64: 62 us so, 71 without; 8,192 x 8,
// D 128: 270 / 309; 2 x 2,048 x 8, D 256: 139 / 161).
// Parts that all fit then go to the first workgroups: with empty ones in between, the shader engines, which are dealt
// workgroups in turn, get unequal work (20 rows of 16 sequences x 8 heads, D 128, every other one 64 tokens long, the
// others 4,096: 38 us, 58 with empty ones in between).  Tiles of prompts keep their place instead, heaviest first over all
// sequences (2 x 4,096 tokens: 89 us, 101 sequence by sequence).  So do those of bounds that descend: segments that share
// rows can have more tiles than the grid, and the join would read parts that no workgroup has written.
// Every workgroup computes the same sums in the same order.
struct PagedPlanCall {   // the same in all of a call's workgroups
  PagedDiv G;            // query heads of a key head
  int rows, Hk;          // rows of a tile; key heads
  int splits, least, slots;
  int64_t tiles;
  bool causal;
};
struct PagedPlanSeg {    // what a segment brings (a lane has one)
  PagedSeg seg;
  int tiles, blocks, unseen;
  bool descends;         // its bounds do
};
POPE_HD PagedPlanSeg paged_plan_seg(const PagedSeqs& q, const PagedPlanCall& c, int s) {
  PagedPlanSeg p = {};
  if (s < (q.cu ? q.B + 2 : q.B)) {
    p.seg = paged_seg(q, s);
    p.descends = q.cu && paged_bound(q, s) > paged_bound(q, s + 1);
    p.tiles = (int)(((int64_t)p.seg.n * c.G.d + c.rows - 1) / c.rows);
    p.blocks = (p.seg.len + kBlockKeys - 1) / kBlockKeys;
    const int rows = p.seg.n / kBlockKeys;
    p.unseen = c.causal ? (rows < p.blocks ? rows : p.blocks) / 4 : 0;
  }
  return p;
}
// Workgroup `at` of a key head (split * tiles + tile, tiles in reverse: later ones see the most keys when causal).
struct PagedPlan { PagedTile t; int tile, split, least; bool dealt; };
// The wave: sum(f), any(f) and all(f) over its 64 segments; first_above(f, at): the first one whose sum of f up to and with it
// exceeds `at`, and that sum without it (64: none does); of(i, f): f of the i-th; hits: as above.
template <typename Wave>
POPE_HD PagedPlan paged_plan_of(const PagedSeqs& q, const PagedPlanCall& c, int at, const Wave& w) {
  PagedPlan r;
  const unsigned n = (unsigned)c.tiles;
  r.split = (int)((unsigned)at / n);
  r.tile = (int)(n - 1 - ((unsigned)at - (unsigned)r.split * n));
  r.least = c.least;
  r.dealt = false;
  if (c.slots) {
    const float slots = (float)c.slots / (float)c.Hk;
    const auto each = [](const PagedPlanSeg& s) { return (float)(s.blocks - s.unseen); };
    // 2^26 blocks: all positions
    const float even = __builtin_ceilf(w.sum([&](const PagedPlanSeg& s) { return (float)s.tiles * each(s); }) / slots);
    const int cut = (int)(even < 67108864.f ? even : 67108864.f);
    int least = c.least > cut ? c.least : cut;
    bool fits = false;
    for (int i = 0; i < 16 && !fits; ++i) {
      fits = w.sum([&](const PagedPlanSeg& s) {
        const float parts = __builtin_ceilf(each(s) / (float)least);
        return (float)s.tiles * (parts > 1.f ? parts : 1.f);
      }) <= slots;
      if (!fits) least += least / 16 > 1 ? least / 16 : 1;
    }
    r.least = least;
    if (fits && !w.any([](const PagedPlanSeg& s) { return s.descends || (s.tiles > 1 && s.blocks > 0 && 8 * s.unseen >= s.blocks); })) {
      const auto parts = [&](const PagedPlanSeg& s) {
        const int p = (s.blocks + least - 1) / least, m = p < c.splits ? p : c.splits;
        return m > 1 ? m : 1;
      };
      int before;
      const int f = w.first_above([&](const PagedPlanSeg& s) { return s.tiles * parts(s); }, at, &before);
      r.dealt = true;
      r.t.seg = PagedSeg{-1, 0, 0, 0, 0, 0};
      r.t.local = r.split = r.tile = 0;
      r.least = 1;
      if (f == 64) return r;
      const int count = w.of(f, [](const PagedPlanSeg& s) { return s.tiles; }), k = at - before;
      r.split = k / count;
      r.t.seg = PagedSeg{w.of(f, [](const PagedPlanSeg& s) { return s.seg.b; }),    w.of(f, [](const PagedPlanSeg& s) { return s.seg.batch; }),
                         w.of(f, [](const PagedPlanSeg& s) { return s.seg.row0; }), w.of(f, [](const PagedPlanSeg& s) { return s.seg.n; }),
                         w.of(f, [](const PagedPlanSeg& s) { return s.seg.len; }),  w.of(f, [](const PagedPlanSeg& s) { return s.seg.first; })};
      r.t.local = count - 1 - (k - r.split * count);
      r.tile = q.cu ? (int)paged_first_tile(q, f, c.G.d, c.rows, 1) + r.t.local : r.t.local * q.B + f;
      const int same = w.of(f, [&](const PagedPlanSeg& s) { const int p = parts(s); return (s.blocks + p - 1) / p; });   // a sequence's parts alike
      r.least = same > 1 ? same : 1;
      return r;
    }
  }
  r.t = paged_tile_of(q, r.tile, c.G.d, c.rows, 1, w);
  return r;
}

// Rows of a tile that starts at row r0 of its segment: row r0 + x is query head g Hk + hk of new token i, r = i G + g.
struct PagedRowMap {
  unsigned i0, rem, G;
  PagedDiv div;
  POPE_HD PagedRowMap(int r0, const PagedDiv& g) : i0(g.of(r0)), rem(r0 - i0 * g.d), G(g.d), div(g) {}
  POPE_HD int token(int x) const { return (int)(i0 + div.of(rem + x)); }
  POPE_HD int group(int x) const { return (int)(rem + x - div.of(rem + x) * G); }
};

// Blocks of keys a tile's rows see, over all of them.
POPE_HD int paged_tile_blocks(const PagedSeg& g, int local, int rows, const PagedDiv& G, bool causal) {
  const int64_t all = (int64_t)g.n * G.d, end = (int64_t)(local + 1) * rows;
  const int last = (int)(end < all ? end : all) - 1;
  const int limit = last < local * rows ? 0 : paged_limit(g.first + (int)G.of(last), g.len, causal);
  return (limit + kBlockKeys - 1) / kBlockKeys;
}

// Layout of a (page, head): blocks of 32 slots, each in the operand order of the 16x16x32 MFMAs that read it,
// so that a wave's load is 64 lanes x 16 consecutive bytes and no operand passes through LDS.
//   K (A operand, rows = keys, k = columns): step e / 32, key half t / 16, lane t % 16 + 16 (e % 32 / 8), element e % 8
//   V (A operand, rows = columns, k = keys): tile d / 16, lane d % 16 + 16 (t % 16 / 4), element 4 (t / 16) + t % 4:
//     the order in which the two 16-key score tiles of a block hold their keys, so P needs no shuffle
// 16-bit: one MFMA operand per 16 bytes of a lane.  8-bit: two of 8 bytes each (K: both key halves, V: tiles 2 v, 2 v + 1).
// steps = k steps of 32 columns, tiles = V tiles of 16 columns (even).  Offsets in elements.
POPE_HD int paged_k_off(bool q8, int t, int e) {
  const int step = e >> 5, half = t >> 4, lane = (t & 15) + 16 * ((e & 31) >> 3), j = e & 7;
  return q8 ? ((step * 64 + lane) * 2 + half) * 8 + j : ((step * 2 + half) * 64 + lane) * 8 + j;
}
POPE_HD int paged_v_off(bool q8, int t, int d) {
  const int tile = d >> 4, lane = (d & 15) + 16 * ((t & 15) >> 2), j = 4 * (t >> 4) + (t & 3);
  return q8 ? (((tile >> 1) * 64 + lane) * 2 + (tile & 1)) * 8 + j : (tile * 64 + lane) * 8 + j;
}
// Exponent byte of slot t (which = 0: K, 1: V) in the block's 64: four keys' K bytes, then their V bytes, so that a lane
// reads those of its four score rows at once.
POPE_HD int paged_scale_off(int t, int which) { return (t >> 2) * 8 + which * 4 + (t & 3); }

// k steps and V tiles of a head: the instances the kernels are built for.
POPE_HD int paged_v_tiles(int D) { return D <= 32 ? 2 : D <= 64 ? 4 : D <= 96 ? 6 : D <= 128 ? 8 : 16; }
POPE_HD int paged_k_steps(int D, int R) {
  const int tiles = paged_v_tiles(D), need = (D + R + 31) / 32;
  const int half = tiles / 2, mid = (3 * tiles + 3) / 4;
  return need <= half ? half : need <= mid ? mid : tiles;
}

}  // namespace pope
