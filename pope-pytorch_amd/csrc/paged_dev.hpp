// Device helpers of the paged cache's kernels.
#pragma once
#include "paged.hpp"
#include "pope_common.hpp"

namespace pope {

// The segment that tile `tile` belongs to, and its tile within it; seg.n = 0 where there is none.  Packed calls: the
// lanes of a wave test 64 segments' first tiles at a time, the last one at or below `tile` has it (with bounds that
// decrease, any segment may come out, and paged_seg bounds it).  Padded calls: the sequences' n-th tiles side by side.
struct PagedTile { PagedSeg seg; int local; };
__device__ __forceinline__ PagedTile paged_tile(const PagedSeqs& q, int tile, int unit, int per, int extra) {
  PagedTile t;
  if (!q.cu) {
    t.local = (int)((unsigned)tile / (unsigned)q.B);
    t.seg = paged_seg(q, tile - t.local * q.B);
    return t;
  }
  const int lane = threadIdx.x & 63, S = q.B + 2;
  int found = 0;
  for (int s0 = 0; s0 < S; s0 += 64) {
    const int s = s0 + lane;
    const bool at = s < S && paged_first_tile(q, s < S ? s : 0, unit, per, extra) <= tile;
    const uint64_t w = __ballot(at);
    if (!w) break;
    found = s0 + 63 - __builtin_clzll(w);
    if (found != s0 + 63) break;
  }
  found = __builtin_amdgcn_readfirstlane(found);
  t.seg = paged_seg(q, found);
  t.local = tile - paged_first_tile(q, found, unit, per, extra);
  return t;
}

// Page of block `blk` of sequence b; -1 for a number outside the cache.
__device__ __forceinline__ int paged_page(const PagedCache& c, int b, int blk) {
  const int id = c.table[(int64_t)b * c.table_sb + (blk >> c.blk_shift)];
  return (unsigned)id < (unsigned)c.pages ? id : -1;
}
// Elements before block `blk` of (page, head h) in the K or V pages (`head`: elements of a (page, head)).
__device__ __forceinline__ int64_t paged_block_off(const PagedCache& c, int page, int h, int blk, int64_t head, int elems) {
  const int sub = blk & ((1 << c.blk_shift) - 1);
  return ((int64_t)page * c.Hk + h) * head + (int64_t)sub * elems;
}
__device__ __forceinline__ int64_t paged_scale_base(const PagedCache& c, int page, int h, int blk) {
  const int sub = blk & ((1 << c.blk_shift) - 1);
  return ((((int64_t)page * c.Hk + h) << c.blk_shift) + sub) * 64;
}

// Eight e4m3 codes -> a 16-bit MFMA operand: codes have 4 significant bits and magnitudes 2^-9 .. 448, so both types hold
// them exactly; times `unit` (a power of two) bf16 does too.
template <typename T>
__device__ __forceinline__ u32x4 unpack_e4m3(u32x2 w, float unit) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (T::kCode == 2) {
      r[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], unit, false));
      r[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], unit, true));
    } else {
      r[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], unit, false));
      r[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], unit, true));
    }
  }
  return r;
}

// Workgroup -> (key head, row tile, split): heads fastest, so that a head's tiles, which read the same keys, run at once
// on one XCD (ids are dealt round-robin to the 8 XCDs); later tiles first, which see the most keys when causal.
struct PagedJob { int tile, hk, split; };
__device__ __forceinline__ PagedJob paged_job(const PagedAttnParams& p) {
  const unsigned id = blockIdx.x, rest = id / (unsigned)p.c.Hk, n = (unsigned)p.tiles, split = rest / n, x = rest - split * n;
  return PagedJob{(int)(n - 1 - x), (int)(id - rest * p.c.Hk), (int)split};
}

// A workgroup's tile, part of the key axis, and the least blocks of a part.
//
// Many rows, at most 64 segments (`slots`, the workgroups that the chip holds, is not 0): parts are cut by what the sequences
// have, as few blocks as these workgroups get of all tiles' blocks, or more where the tiles' parts would then be more
// than the workgroups.  A quarter of what causality takes from a prompt's first rows is left out: its heaviest tile has
// twice the mean's blocks and would end alone (prompts of 4,096 tokens x 8 heads, D 64: 62 us so, 71 without; 8,192 x 8,
// D 128: 270 / 309; 2 x 2,048 x 8, D 256: 139 / 161).
// Parts that all fit then go to the first workgroups: with empty ones in between, the shader engines, which are dealt
// workgroups in turn, get unequal work (20 rows of 16 sequences x 8 heads, D 128, every other one 64 tokens long, the
// others 4,096: 38 us, 58 with empty ones in between).  Tiles of prompts keep paged_job's order instead, heaviest first
// over all sequences (2 x 4,096 tokens: 89 us, 101 sequence by sequence).
// Every workgroup computes the same sums in the same order.
struct PagedPlan { PagedTile t; int tile, hk, split, least; };
__device__ __forceinline__ PagedPlan paged_plan(const PagedAttnParams& p, int rows) {
  const PagedSeqs& q = p.c.seqs;
  const PagedJob job = paged_job(p);
  PagedPlan r;
  r.tile = job.tile;
  r.hk = job.hk;
  r.split = job.split;
  r.least = p.least;
  if (p.slots) {
    const int s = threadIdx.x & 63;
    PagedSeg g = {};
    int tiles = 0, blocks = 0, unseen = 0;
    if (s < (q.cu ? q.B + 2 : q.B)) {
      g = paged_seg(q, s);
      tiles = (int)(((int64_t)g.n * p.G.d + rows - 1) / rows);
      blocks = (g.len + kBlockKeys - 1) / kBlockKeys;
      unseen = p.causal ? min(g.n / kBlockKeys, blocks) / 4 : 0;
    }
    auto sum = [](float x) {
#pragma unroll
      for (int i = 1; i < 64; i *= 2) x += wave_shfl_xor(x, i);
      return x;
    };
    const float slots = (float)p.slots / (float)p.c.Hk, n = (float)tiles, each = (float)(blocks - unseen);
    int least = max(p.least, (int)fminf(__builtin_ceilf(sum(n * each) / slots), 67108864.f));   // 2^26 blocks: all positions
    bool fits = false;
    for (int i = 0; i < 16 && !fits; ++i) {
      fits = sum(n * fmaxf(1.f, __builtin_ceilf(each / (float)least))) <= slots;
      if (!fits) least += max(1, least / 16);
    }
    r.least = __builtin_amdgcn_readfirstlane(least);
    if (__builtin_amdgcn_readfirstlane(fits) && !__any(tiles > 1 && 8 * unseen >= blocks)) {
      const int parts = max(1, min(p.splits, (blocks + r.least - 1) / r.least)), mine = tiles * parts;
      int upto = mine;
#pragma unroll
      for (int i = 1; i < 64; i *= 2) {
        const int x = __shfl_up(upto, i, 64);
        upto += s >= i ? x : 0;
      }
      const int at = (int)(blockIdx.x / (unsigned)p.c.Hk);
      const uint64_t behind = __ballot(upto > at);
      const int f = behind ? __builtin_ctzll(behind) : 0;
      auto of = [&](int x) { return __builtin_amdgcn_readlane(x, f); };
      r.t.seg = PagedSeg{of(g.b), of(g.batch), of(g.row0), behind ? of(g.n) : 0, of(g.len), of(g.first)};
      const int count = max(of(tiles), 1), k = at - (of(upto) - of(mine));
      r.split = behind ? k / count : 0;
      r.t.local = behind ? count - 1 - (k - r.split * count) : 0;
      r.least = max(1, of((blocks + parts - 1) / parts));   // a sequence's parts alike
      r.tile = q.cu ? (int)paged_first_tile(q, f, p.G.d, rows, 1) + r.t.local : r.t.local * q.B + f;
      return r;
    }
  }
  r.t = paged_tile(q, job.tile, p.G.d, rows, 1);
  return r;
}

// Rows of a tile that starts at row r0 of its segment: row r0 + x is query head g Hk + hk of new token i, r = i G + g.
struct PagedRowMap {
  unsigned i0, rem, G;
  PagedDiv div;
  __device__ __forceinline__ PagedRowMap(int r0, const PagedDiv& g) : i0(g.of(r0)), rem(r0 - i0 * g.d), G(g.d), div(g) {}
  __device__ __forceinline__ int token(int x) const { return (int)(i0 + div.of(rem + x)); }
  __device__ __forceinline__ int group(int x) const { return (int)(rem + x - div.of(rem + x) * G); }
};

// Q_hat of a tile's rows, eight columns of a row at a time: their inputs, loaded ahead; made and stored as the sum of two
// 16-bit parts each; and the zeros behind a row.
struct PagedQueryIn {
  u32x4 x;        // the queries
  f32x4 f[2];     // their angles
};
template <typename T>
__device__ __forceinline__ PagedQueryIn paged_query_load(const PagedAttnParams& p, const PagedSeg& g, const PagedRowMap& map, int x, int count, int hk, int d0) {
  const PagedCache& c = p.c;
  PagedQueryIn in;
  in.x = u32x4{0, 0, 0, 0};
  in.f[0] = in.f[1] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (x >= count || d0 >= c.D) return in;
  const unsigned r = map.rem + x, i = map.div.of(r), gi = r - i * map.G;
  const int64_t tok = g.row0 + (int)(map.i0 + i);
  const uint16_t* src = p.q + (int64_t)g.batch * p.q_s[0] + (int64_t)(gi * c.Hk + hk) * p.q_s[1] + tok * p.q_s[2] + d0;
  if (p.q_vec) {   // D a multiple of 8, rows 16-byte aligned
    in.x = *reinterpret_cast<const u32x4*>(src);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (d0 + k < c.D) in.x[k >> 1] |= (uint32_t)src[k] << (16 * (k & 1));
  }
  if (d0 < c.R) {
    const float* fr = p.freqs + (int64_t)g.batch * p.f_s[0] + tok * p.f_s[1] + d0;
    if (p.f_vec) {   // R a multiple of 8, rows 16-byte aligned
      in.f[0] = *reinterpret_cast<const f32x4*>(fr);
      in.f[1] = *reinterpret_cast<const f32x4*>(fr + 4);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (d0 + k < c.R) in.f[k >> 2][k & 3] = fr[k];
    }
  }
  return in;
}
// Rows past the tile's are softplus(0) cos 0, or zeros where all of a wave's are (`live`): finite values that nothing reads.
template <typename T>
__device__ __forceinline__ void paged_query_make(const PagedAttnParams& p, const PagedQueryIn& in, bool live, int row, int d0, int stride, uint16_t* hi, uint16_t* lo) {
  const int D = p.c.D, R = p.c.R;
  if (d0 >= D) return;
  float x[8], a[8], b[8];   // a: cosine part, or the raw value; b: sine part
  unpack8<T>(in.x, x);
  const bool off = p.q_factor == 0.f;   // scores are 0, also of values that are not finite
  if (!live) {
#pragma unroll
    for (int k = 0; k < 8; ++k) a[k] = b[k] = 0.f;
  } else if (d0 < R) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float sn, cs;
      sincos_rev(in.f[k >> 2][k & 3], &sn, &cs);
      const float m = softplus_f(x[k]) * p.q_factor;
      const bool rot = d0 + k < R;
      a[k] = off ? 0.f : rot ? m * cs : x[k] * p.q_factor;
      b[k] = off ? 0.f : m * sn;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) a[k] = off ? 0.f : x[k] * p.q_factor;
  }
  auto store = [&](int e, const float* v) {   // eight columns from e on
    u32x4 wh, wl;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      wh[k] = T::pack2(v[2 * k], v[2 * k + 1]);
      wl[k] = T::pack2(v[2 * k] - T::to_float((uint16_t)wh[k]), v[2 * k + 1] - T::to_float((uint16_t)(wh[k] >> 16)));
    }
    *reinterpret_cast<u32x4*>(hi + row * stride + e) = wh;
    *reinterpret_cast<u32x4*>(lo + row * stride + e) = wl;
  };
  if (R % 8 == 0) {   // a chunk is all rotated or all not, and its columns start on a chunk
    if (d0 < R) store(d0, a), store(R + d0, b);
    else store(R + d0, a);
  } else {
    auto put = [&](int e, float v) {
      const uint16_t w = T::bits(v);
      hi[row * stride + e] = w;
      lo[row * stride + e] = T::bits(v - T::to_float(w));
    };
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int d = d0 + k;
      if (d >= D) break;
      put(d < R ? d : R + d, a[k]);
      if (d < R) put(R + d, b[k]);
    }
  }
}
template <int ROWS>
__device__ __forceinline__ void paged_query_tail(const PagedAttnParams& p, int at, int n, int cols, int stride, uint16_t* hi, uint16_t* lo) {
  const int D = p.c.D, R = p.c.R, E = R % 8 == 0 ? R + (D + 7) / 8 * 8 : D + R;
  for (int it = at; it < ROWS * (cols - E); it += n) hi[it % ROWS * stride + E + it / ROWS] = lo[it % ROWS * stride + E + it / ROWS] = 0;
}

// Blocks of keys a tile's rows see, over all of them.
__device__ __forceinline__ int paged_tile_blocks(const PagedSeg& g, int local, int rows, const PagedDiv& G, bool causal) {
  const int last = min((local + 1) * rows, g.n * (int)G.d) - 1;
  const int limit = last < local * rows ? 0 : paged_limit(g.first + (int)G.of(last), g.len, causal);
  return (limit + kBlockKeys - 1) / kBlockKeys;
}

template <typename T>
__device__ __forceinline__ bool nonfinite16(uint32_t bits) {
  constexpr uint32_t e = T::kCode == 2 ? 0x7f80u : 0x7c00u;
  return (bits & e) == e;
}

}  // namespace pope
