// Device helpers of the paged cache's kernels.
#pragma once
#include "paged.hpp"
#include "pope_common.hpp"

namespace pope {

// A wave's lanes as the segments that paged_index.hpp's functions go over.
struct PagedWave {
  PagedPlanSeg mine;
  template <typename F>
  __device__ __forceinline__ uint64_t operator()(F&& f) const { return __ballot(f((int)(threadIdx.x & 63))); }
  template <typename F>
  __device__ __forceinline__ float sum(F&& f) const {
    float x = f(mine);
#pragma unroll
    for (int i = 1; i < 64; i *= 2) x += wave_shfl_xor(x, i);
    return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x)));
  }
  template <typename F>
  __device__ __forceinline__ bool any(F&& f) const { return __any(f(mine)); }
  template <typename F>
  __device__ __forceinline__ int of(int i, F&& f) const { return __builtin_amdgcn_readlane(f(mine), i); }
  template <typename F>
  __device__ __forceinline__ int first_above(F&& f, int at, int* before) const {
    const int lane = threadIdx.x & 63, own = f(mine);
    int upto = own;
#pragma unroll
    for (int i = 1; i < 64; i *= 2) {
      const int x = __shfl_up(upto, i, 64);
      upto += lane >= i ? x : 0;
    }
    const uint64_t above = __ballot(upto > at);
    const int i = above ? __builtin_ctzll(above) : 64;
    *before = above ? __builtin_amdgcn_readlane(upto - own, i) : 0;
    return i;
  }
};
__device__ __forceinline__ PagedTile paged_tile(const PagedSeqs& q, int tile, int unit, int per, int extra) {
  return paged_tile_of(q, tile, unit, per, extra, PagedWave{});
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

__device__ __forceinline__ PagedPlan paged_plan(const PagedAttnParams& p, int rows) {
  const PagedPlanCall call{p.G, rows, p.c.Hk, p.splits, p.least, p.slots, p.tiles, p.causal != 0};
  PagedWave w{};
  if (p.slots) w.mine = paged_plan_seg(p.c.seqs, call, threadIdx.x & 63);
  return paged_plan_of(p.c.seqs, call, (int)(blockIdx.x / (unsigned)p.c.Hk), w);
}

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
      a[k] = rot ? m * cs : x[k] * p.q_factor;
      b[k] = m * sn;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) a[k] = x[k] * p.q_factor;
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

template <typename T>
__device__ __forceinline__ bool nonfinite16(uint32_t bits) {
  constexpr uint32_t e = T::kCode == 2 ? 0x7f80u : 0x7c00u;
  return (bits & e) == e;
}

__device__ __forceinline__ bool finite_f(float x) { return fabsf(x) <= 3.402823466e38f; }

// An average of values, as it goes out: fp16's stay finite where the values were.  A value of an 8-bit page may stand for 65536
// (it is read as 65504 too), and P is rounded where its sum is not, which may carry an average up to 2^-11 past the values.
template <typename T>
__device__ __forceinline__ f32x4 averages(f32x4 x) {
  if constexpr (T::kCode == 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = finite_f(x[i]) ? fminf(fmaxf(x[i], -65504.f), 65504.f) : x[i];
  }
  return x;
}

// Rows that are NaN although their queries are not: infinite keys and values.  Products of a sum of two 16-bit parts, or of
// a P that is 0 in 16 bits, turn an infinity into NaN (hi x inf + lo x inf; 0 x inf) where the formula has +-inf, or a score
// of -inf and so a weight of 0.  The loops do not look for that: a wave (many rows: a workgroup) that ends with such rows goes
// over its blocks a second time, with the finite elements of K times both parts, the others times the signs of Q_hat, and V's
// others outside the product, as in blocks with keys that some row does not see.  What is finite goes through the same
// operations in the same order, so the other rows keep their bits.  (A query column that 16 bits round to 0 counts as 0, as
// does a weight that fp32 does; a row whose values or keys hold a NaN that it sees is computed twice and stays NaN.)  8-bit
// pages hold no infinity.
//
// A 16-bit operand's finite elements, and the others; zeros in the places of either's rest.
template <typename T>
__device__ __forceinline__ void split_finite(u32x4 w, u32x4* fin, u32x4* rest) {
  constexpr uint32_t kOne = T::kCode == 2 ? 0x00800080u : 0x04000400u;   // carries into the sign where all exponent bits are set
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t m = ((((w[i] & 0x7fff7fffu) + kOne) & 0x80008000u) >> 15) * 0xffffu;
    (*fin)[i] = w[i] & ~m;
    (*rest)[i] = w[i] & m;
  }
}
// The signs of an operand's elements: -1, 0 or 1.
template <typename T>
__device__ __forceinline__ typename T::vec8 sign_operand(typename T::vec8 q) {
  constexpr uint32_t kUnit = T::kCode == 2 ? 0x3f803f80u : 0x3c003c00u;
  u32x4 w = __builtin_bit_cast(u32x4, q);
  asm volatile("" : "+v"(w));   // made where it is used, not in front of the loop
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = ((w[i] & 0x80008000u) | kUnit) & (((((w[i] & 0x7fff7fffu) + 0x7fff7fffu) & 0x80008000u) >> 15) * 0xffffu);
  return as_vec8<typename T::vec8>(w);
}
template <typename T>
__device__ __forceinline__ bool all_finite(typename T::vec8 q) {
  u32x4 fin, rest;
  split_finite<T>(__builtin_bit_cast(u32x4, q), &fin, &rest);
  return (rest[0] | rest[1] | rest[2] | rest[3]) == 0;
}

// A 16-byte unit of values, of which the first keys below `have` are there (key 16 (j / 4) + j % 4 for element j of a 16-bit
// unit; 8-bit: two units of 8): the others and what is not finite become zeros, and the latter's keys are noted in `odd`
// (at `key0` in the block).
template <typename T, bool Q8>
__device__ __forceinline__ void clean_values(u32x4& w, int have, int key0, uint32_t& odd) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t keep = 0;
#pragma unroll
    for (int e = 0; e < (Q8 ? 4 : 2); ++e) {
      const int j = Q8 ? (4 * i + e) & 7 : 2 * i + e, key = 16 * (j >> 2) + (j & 3), sh = (Q8 ? 8 : 16) * e;
      const uint32_t x = w[i] >> sh;
      const bool there = key < have, fin = Q8 ? (x & 0x7f) != 0x7f : !nonfinite16<T>(x);
      keep |= there && fin ? (Q8 ? 0xffu : 0xffffu) << sh : 0u;
      odd |= there && !fin ? 1u << (key + key0) : 0u;
    }
    w[i] &= keep;
  }
}

}  // namespace pope
