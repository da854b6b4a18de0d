// Device helpers of the paged cache's kernels.
#pragma once
#include "paged.hpp"
#include "pope_common.hpp"

namespace pope {

// The segment that tile `tile` belongs to, and its tile within it; seg.n = 0 where there is none.  Packed calls: the
// lanes of a wave test 64 segments' first tiles at a time, the last one at or below `tile` has it (with bounds that
// decrease, any segment may come out, and paged_seg bounds it).
struct PagedTile { PagedSeg seg; int64_t local; };
__device__ __forceinline__ PagedTile paged_tile(const PagedSeqs& q, int64_t tile, int unit, int per, int extra) {
  PagedTile t;
  if (!q.cu) {
    const int64_t each = ((int64_t)q.N * unit + per - 1) / per + extra - 1;
    const int b = (int)(tile / each);
    t.seg = paged_seg(q, b);
    t.local = tile - (int64_t)b * each;
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

// Eight e4m3 codes -> a 16-bit MFMA operand (exact: at most 4 significant bits, magnitudes 2^-9 .. 448).
template <typename T>
__device__ __forceinline__ u32x4 unpack_e4m3(u32x2 w) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (T::kCode == 2) {
      r[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], 1.f, false));
      r[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], 1.f, true));
    } else {
      r[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], 1.f, false));
      r[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], 1.f, true));
    }
  }
  return r;
}

}  // namespace pope
