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
