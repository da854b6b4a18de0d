// Device helpers of the paged cache's kernels.
#pragma once
#include "paged.hpp"
#include "pope_common.hpp"

namespace pope {

// The segment that tile `tile` belongs to, and its tile within it; seg.n = 0 where there is none.  Packed calls: the
// lanes of a wave test 64 segments' first tiles at a time, the last one at or below `tile` has it (with bounds that
// decrease, any segment may come out, and paged_seg bounds it).  Padded calls: the sequences' n-th tiles side by side.
struct PagedTile { PagedSeg seg; int64_t local; };
__device__ __forceinline__ PagedTile paged_tile(const PagedSeqs& q, int64_t tile, int unit, int per, int extra) {
  PagedTile t;
  if (!q.cu) {
    t.local = tile / q.B;
    t.seg = paged_seg(q, (int)(tile - t.local * q.B));
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
struct PagedJob { int64_t tile; int hk, split; };
__device__ __forceinline__ PagedJob paged_job(const PagedAttnParams& p) {
  const int64_t id = blockIdx.x, rest = id / p.c.Hk;
  return PagedJob{p.tiles - 1 - rest % p.tiles, (int)(id - rest * p.c.Hk), (int)(rest / p.tiles)};
}

// Rows of a tile that starts at row r0 of its segment: row r0 + x is query head g Hk + hk of new token i, r = i G + g.
struct PagedRowMap {
  int i0, rem, G;
  __device__ __forceinline__ PagedRowMap(int64_t r0, int g) : i0((int)(r0 / g)), rem((int)(r0 - (int64_t)i0 * g)), G(g) {}
  __device__ __forceinline__ int token(int x) const { return i0 + (int)((unsigned)(rem + x) / (unsigned)G); }
  __device__ __forceinline__ int group(int x) const { return (int)((unsigned)(rem + x) % (unsigned)G); }
};

// Q_hat of `ROWS` rows from x0 on (those below `live`; the others are zeros) by `n` threads, this one the `at`-th, times
// `factor`, each value as the sum of two 16-bit parts; CH columns of a row per thread and turn, all loads independent.
template <typename T, int ROWS, int CH>
__device__ __forceinline__ void paged_query_rows(const PagedAttnParams& p, const PagedSeg& g, const PagedRowMap& map, int x0, int live, int hk,
                                                 int at, int n, int cols, int stride, uint16_t* hi, uint16_t* lo) {
  const PagedCache& c = p.c;
  const int D = c.D, R = c.R, chunks = (D + CH - 1) / CH;
  const bool whole = R % CH == 0;   // a chunk is all rotated or all not, and its columns start on a chunk
  for (int it = at; it < ROWS * chunks; it += n) {
    const int row = it % ROWS, d0 = it / ROWS * CH;
    const bool on = x0 + row < live && p.q_factor != 0.f;
    const int i = g.row0 + (on ? map.token(x0 + row) : 0), h = on ? map.group(x0 + row) * c.Hk + hk : hk;
    const uint16_t* src = p.q + (int64_t)g.batch * p.q_s[0] + (int64_t)h * p.q_s[1] + (int64_t)i * p.q_s[2] + d0;
    const float* fr = p.freqs + (int64_t)g.batch * p.f_s[0] + (int64_t)i * p.f_s[1] + d0;
    float x[CH], f[CH];
    if (p.q_vec) {   // D a multiple of 8, rows 16-byte aligned
      if constexpr (CH == 8) {
        unpack8<T>(on ? *reinterpret_cast<const u32x4*>(src) : u32x4{0, 0, 0, 0}, x);
      } else {
        const u32x2 w = on ? *reinterpret_cast<const u32x2*>(src) : u32x2{0, 0};
#pragma unroll
        for (int k = 0; k < CH; ++k) x[k] = T::to_float((uint16_t)(w[k >> 1] >> (16 * (k & 1))));
      }
    } else {
#pragma unroll
      for (int k = 0; k < CH; ++k) x[k] = on && d0 + k < D ? T::to_float(src[k]) : 0.f;
    }
    if (d0 < R) {
      if (p.f_vec) {   // R a multiple of 8, rows 16-byte aligned
#pragma unroll
        for (int k = 0; k < CH; k += 4) {
          const f32x4 w = on ? *reinterpret_cast<const f32x4*>(fr + k) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int e = 0; e < 4; ++e) f[k + e] = w[e];
        }
      } else {
#pragma unroll
        for (int k = 0; k < CH; ++k) f[k] = on && d0 + k < R ? fr[k] : 0.f;
      }
    }
    float a[CH], b[CH];   // a: cosine part, or the raw value; b: sine part
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      a[k] = x[k] * p.q_factor;
      b[k] = 0.f;
      if (d0 + k < R) {
        float sn, cs;
        sincos_rev(f[k], &sn, &cs);
        const float m = on ? softplus_f(x[k]) * p.q_factor : 0.f;
        a[k] = m * cs;
        b[k] = m * sn;
      }
    }
    auto store = [&](int e, const float* v) {   // CH columns from e on
      uint32_t wh[CH / 2], wl[CH / 2];
#pragma unroll
      for (int k = 0; k < CH / 2; ++k) {
        wh[k] = T::pack2(v[2 * k], v[2 * k + 1]);
        wl[k] = T::pack2(v[2 * k] - T::to_float((uint16_t)wh[k]), v[2 * k + 1] - T::to_float((uint16_t)(wh[k] >> 16)));
      }
#pragma unroll
      for (int k = 0; k < CH / 2; k += 2) {
        *reinterpret_cast<u32x2*>(hi + row * stride + e + 2 * k) = u32x2{wh[k], wh[k + 1]};
        *reinterpret_cast<u32x2*>(lo + row * stride + e + 2 * k) = u32x2{wl[k], wl[k + 1]};
      }
    };
    if (whole) {
      if (d0 < R) {
        store(d0, a);
        store(R + d0, b);
      } else {
        store(R + d0, a);
      }
    } else {
      auto put = [&](int e, float v) {
        const uint16_t w = T::bits(v);
        hi[row * stride + e] = w;
        lo[row * stride + e] = T::bits(v - T::to_float(w));
      };
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        const int d = d0 + k;
        if (d >= D) break;
        put(d < R ? d : R + d, a[k]);
        if (d < R) put(R + d, b[k]);
      }
    }
  }
  const int E = whole ? R + chunks * CH : D + R;
  for (int it = at; it < ROWS * (cols - E); it += n) hi[it % ROWS * stride + E + it / ROWS] = lo[it % ROWS * stride + E + it / ROWS] = 0;
}

// Blocks of keys a tile's rows see, over all of them.
__device__ __forceinline__ int paged_tile_blocks(const PagedSeg& g, int64_t local, int rows, int G, bool causal) {
  const int64_t all = (int64_t)g.n * G, end = (local + 1) * rows;
  const int64_t last = (end < all ? end : all) - 1;
  const int limit = last < local * rows ? 0 : paged_limit(g.first + (int)(last / G), g.len, causal);
  return (limit + kBlockKeys - 1) / kBlockKeys;
}

// x with the 16-bit (8-bit) elements j of which (keep >> j) & 1 is 0 cleared.
__device__ __forceinline__ u32x4 keep16(u32x4 x, uint32_t keep) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] &= ((keep >> (2 * i)) & 1 ? 0xffffu : 0u) | ((keep >> (2 * i + 1)) & 1 ? 0xffff0000u : 0u);
  return x;
}

template <typename T>
__device__ __forceinline__ bool nonfinite16(uint32_t bits) {
  constexpr uint32_t e = T::kCode == 2 ? 0x7f80u : 0x7c00u;
  return (bits & e) == e;
}

}  // namespace pope
