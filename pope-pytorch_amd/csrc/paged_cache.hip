// Rows into the paged cache and out of it (gfx950).
//
//   write  K_hat = [softplus(k) cos t, softplus(k) sin t, k], t = F + bias, rounded once: to 16 bits, or to e4m3 codes
//          x 2^-e with one e per (token, head): the smallest with max |x| <= 448 2^e.  A power of two scales exactly, so
//          codes of 16-bit values depend on no rounding but e4m3's own.
//   read   the rows back, K_hat with (cos, sin) pairs interleaved as apply_pope_to_qk lays them out.
//
// A workgroup has the block of 32 slots of one head that a 16-bit MFMA operand spans (paged_index.hpp): rows cross LDS
// between the callers' row order and the pages' operand order, so both sides of the copy are contiguous.  A wave has a
// row at a time: the row's maximum needs no second pass.  Slots of other tokens in the block are not touched: units of
// 16 bytes are stored whole only where all their tokens are written.
//
// The angle is summed and reduced in fp64 (F + bias in fp32 would be off by up to 1e-3 rad at position 32,768) and the
// functions are accurate to about an ulp of fp32, so that a stored value is the rounding of the exact one except next
// to a rounding border.
#include "paged_dev.hpp"

namespace pope {

namespace {

constexpr int kThreads = 256;

// sin and cos of t by Taylor's series after reduction by multiples of pi / 2 in fp64 (|r| <= pi / 4: the first terms
// left out are below 2e-9 and 4e-10).
__device__ __forceinline__ void sincos_wide(double t, float* s, float* c) {
  const double k = __builtin_rint(t * 0.63661977236758134308);
  const float r = (float)__builtin_fma(-k, 1.57079632679489661923, t);
  const int quarter = (int)(long long)k & 3;
  const float z = r * r;
  const float sr = r + r * z * (-1.f / 6 + z * (1.f / 120 + z * (-1.f / 5040 + z * (1.f / 362880))));
  const float cr = 1.f + z * (-0.5f + z * (1.f / 24 + z * (-1.f / 720 + z * (1.f / 40320 + z * (-1.f / 3628800)))));
  const float a = quarter & 1 ? cr : sr, b = quarter & 1 ? sr : cr;
  *s = quarter & 2 ? -a : a;
  *c = (quarter + 1) & 2 ? -b : b;
}

__device__ __forceinline__ float softplus_accurate(float x) { return fmaxf(x, 0.f) + log1pf(expf(-fabsf(x))); }

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) x = fmaxf(x, __shfl_xor(x, k, 64));
  return x;
}

// Biased exponent of the row's power of two.
__device__ __forceinline__ int row_exponent(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, -126), 126) + 127;
}

// What counts for a row's maximum, and what is stored of x: e4m3 has no infinity.
__device__ __forceinline__ bool finite_f(float x) { return fabsf(x) <= 3.402823466e38f; }

// The block's tokens of the call.
struct Block {
  PagedSeg seg;
  int blk;        // block of the sequence's slots; negative: rows without a slot
  int page;       // -1: outside the cache
  int i0;         // row of slot 0 of the block (rows i0 + t, those in [0, n) belong to the call)
  bool any;
};
__device__ __forceinline__ Block find_block(const PagedCache& c, int64_t tile) {
  Block b;
  const PagedTile t = paged_tile(c.seqs, tile, 1, kBlockKeys, 2);
  b.seg = t.seg;
  const int first = floor_div(t.seg.first, kBlockKeys);
  b.blk = first + t.local;
  b.i0 = b.blk * kBlockKeys - t.seg.first;
  b.any = b.i0 < t.seg.n;   // later tiles of the segment are empty
  b.page = b.any && b.blk >= 0 && t.seg.b >= 0 ? paged_page(c, t.seg.b, b.blk) : -1;
  return b;
}

template <typename T, bool Q8, int VT>
__global__ __launch_bounds__(kThreads) void paged_write_kernel(PagedRowsParams p) {
  constexpr int ST = VT * 32 + 1;   // K_hat has at most 2 D columns
  __shared__ float rows[kBlockKeys * ST];
  __shared__ float inv[kBlockKeys];
  const PagedCache& c = p.c;
  const int hk = blockIdx.y, lane = threadIdx.x & 63, wave = wave_id();
  const Block b = find_block(c, blockIdx.x);
  if (!b.any || b.page < 0) return;
  // slots t of the block that the call writes
  auto live = [&](int t) { return (unsigned)(b.i0 + t) < (unsigned)b.seg.n; };
  uint8_t* scales = Q8 ? c.scales + paged_scale_base(c, b.page, hk, b.blk) : nullptr;
  const int D = c.D, R = c.R, E = D + R, KE = c.steps * 32;

  for (int which = 0; which < 2; ++which) {   // keys, then values
    if (which) __syncthreads();
    for (int t = wave; t < kBlockKeys; t += kThreads / 64) {
      float* row = rows + t * ST;
      if (!live(t)) continue;   // (uniform in the wave)
      const int64_t n = b.seg.row0 + b.i0 + t;
      const uint16_t* src = which ? static_cast<const uint16_t*>(p.v) + b.seg.batch * p.v_s[0] + hk * p.v_s[1] + n * p.v_s[2]
                                  : static_cast<const uint16_t*>(p.k) + b.seg.batch * p.k_s[0] + hk * p.k_s[1] + n * p.k_s[2];
      float amax = 0.f;
      auto put = [&](int e, float x) {
        row[e] = x;
        if (Q8 && finite_f(x)) amax = fmaxf(amax, fabsf(x));
      };
      for (int d = lane; d < D; d += 64) {
        const float x = T::to_float(src[d]);
        if (!which && d < R) {
          float sn, cs;
          sincos_wide((double)p.freqs[b.seg.batch * p.f_s[0] + n * p.f_s[1] + d] + (double)p.bias[hk * p.bias_sh + d], &sn, &cs);
          const float m = softplus_accurate(x);
          put(d, m * cs);
          put(R + d, m * sn);
        } else {
          put(which ? d : R + d, x);
        }
      }
      for (int e = (which ? D : E) + lane; e < (which ? VT * 16 : KE); e += 64) row[e] = 0.f;
      if (Q8) {
        const int e = row_exponent(wave_max(amax));
        if (lane == 0) {
          scales[paged_scale_off(t, which)] = (uint8_t)e;
          inv[t] = __uint_as_float((uint32_t)(254 - e) << 23);
        }
      }
    }
    __syncthreads();
    auto at = [&](int t, int e) { return rows[t * ST + e]; };
    auto code = [&](int t, int e) {   // x 2^-e, NaN where x is not finite
      const float x = rows[t * ST + e] * inv[t];
      return finite_f(x) ? x : __builtin_nanf("");
    };
    if (!which) {
      if constexpr (Q8) {
        uint8_t* dst = static_cast<uint8_t*>(c.k) + paged_block_off(c, b.page, hk, b.blk, c.k_head, KE * 32);
        for (int u = threadIdx.x; u < c.steps * 128; u += kThreads) {   // (step, lane, half): 8 bytes
          const int half = u & 1, ln = (u >> 1) & 63, st = u >> 7, t = half * 16 + (ln & 15), e0 = st * 32 + 8 * (ln >> 4);
          if (!live(t)) continue;
          u32x2 w;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            int x = __builtin_amdgcn_cvt_pk_fp8_f32(code(t, e0 + 4 * k), code(t, e0 + 4 * k + 1), 0, false);
            w[k] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(code(t, e0 + 4 * k + 2), code(t, e0 + 4 * k + 3), x, true);
          }
          *reinterpret_cast<u32x2*>(dst + u * 8) = w;
        }
      } else {
        uint16_t* dst = static_cast<uint16_t*>(c.k) + paged_block_off(c, b.page, hk, b.blk, c.k_head, KE * 32);
        for (int u = threadIdx.x; u < c.steps * 128; u += kThreads) {   // (step, half, lane): 16 bytes
          const int ln = u & 63, half = (u >> 6) & 1, st = u >> 7, t = half * 16 + (ln & 15), e0 = st * 32 + 8 * (ln >> 4);
          if (!live(t)) continue;
          u32x4 w;
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = T::pack2(at(t, e0 + 2 * k), at(t, e0 + 2 * k + 1));
          *reinterpret_cast<u32x4*>(dst + u * 8) = w;
        }
      }
      continue;
    }
    // values: a lane's eight elements are eight tokens of one column
    if constexpr (Q8) {
      uint8_t* dst = static_cast<uint8_t*>(c.v) + paged_block_off(c, b.page, hk, b.blk, c.v_head, VT * 512);
      for (int u = threadIdx.x; u < VT * 64; u += kThreads) {   // (tile pair, lane, tile of the pair): 8 bytes
        const int ln = (u >> 1) & 63, d = ((u >> 7) * 2 + (u & 1)) * 16 + (ln & 15), t0 = 4 * (ln >> 4);
        uint32_t w[2];
        bool all = true;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int t = t0 + 16 * k;
          int x = __builtin_amdgcn_cvt_pk_fp8_f32(live(t) ? code(t, d) : 0.f, live(t + 1) ? code(t + 1, d) : 0.f, 0, false);
          w[k] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(live(t + 2) ? code(t + 2, d) : 0.f, live(t + 3) ? code(t + 3, d) : 0.f, x, true);
          all = all && live(t) && live(t + 3);
        }
        if (all) {
          *reinterpret_cast<u32x2*>(dst + u * 8) = u32x2{w[0], w[1]};
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (live(t0 + 16 * (j >> 2) + (j & 3))) dst[u * 8 + j] = (uint8_t)(w[j >> 2] >> (8 * (j & 3)));
        }
      }
    } else {
      uint16_t* dst = static_cast<uint16_t*>(c.v) + paged_block_off(c, b.page, hk, b.blk, c.v_head, VT * 512);
      for (int u = threadIdx.x; u < VT * 64; u += kThreads) {   // (tile, lane): 16 bytes
        const int ln = u & 63, d = (u >> 6) * 16 + (ln & 15), t0 = 4 * (ln >> 4);
        uint16_t w[8];
        bool all = true;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int t = t0 + 16 * (j >> 2) + (j & 3);
          all = all && live(t);
          w[j] = live(t) ? T::bits(at(t, d)) : (uint16_t)0;
        }
        if (all) {
          u32x4 x;
#pragma unroll
          for (int k = 0; k < 4; ++k) x[k] = w[2 * k] | ((uint32_t)w[2 * k + 1] << 16);
          *reinterpret_cast<u32x4*>(dst + u * 8) = x;
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (live(t0 + 16 * (j >> 2) + (j & 3))) dst[u * 8 + j] = w[j];
        }
      }
    }
  }
}

// A dequantised value in the 16-bit type; fp16 has no value above 65504 (a code may round up to one).
template <typename T>
__device__ __forceinline__ uint16_t value_bits(float x) {
  if (T::kCode == 1 && finite_f(x)) x = fminf(fmaxf(x, -65504.f), 65504.f);
  return T::bits(x);
}

template <typename T, bool Q8, int VT>
__global__ __launch_bounds__(kThreads) void paged_read_kernel(PagedRowsParams p) {
  constexpr int ST = VT * 32 + 2;
  __shared__ uint16_t rows[kBlockKeys * ST];
  const PagedCache& c = p.c;
  const int hk = blockIdx.y, lane = threadIdx.x & 63, wave = wave_id();
  const Block b = find_block(c, blockIdx.x);
  if (!b.any) return;
  auto live = [&](int t) { return (unsigned)(b.i0 + t) < (unsigned)b.seg.n; };
  const uint8_t* scales = Q8 && b.page >= 0 ? c.scales + paged_scale_base(c, b.page, hk, b.blk) : nullptr;
  const int D = c.D, R = c.R, E = D + R, KE = c.steps * 32;
  auto scale = [&](int t, int which) { return (int)scales[paged_scale_off(t, which)] - 127; };
  auto code_at = [&](u32x2 w, int j) {
    const uint32_t x = w[j >> 2] >> (8 * (j & 3));
    return __builtin_amdgcn_cvt_f32_fp8((int)x, 0);
  };

  for (int which = 0; which < 2; ++which) {
    if (which) __syncthreads();
    if (b.page >= 0) {
      if (!which) {
        const char* src = static_cast<const char*>(c.k) + paged_block_off(c, b.page, hk, b.blk, c.k_head, KE * 32) * (Q8 ? 1 : 2);
        for (int u = threadIdx.x; u < c.steps * 128; u += kThreads) {
          if constexpr (Q8) {
            const int half = u & 1, ln = (u >> 1) & 63, st = u >> 7, t = half * 16 + (ln & 15), e0 = st * 32 + 8 * (ln >> 4);
            const u32x2 w = *reinterpret_cast<const u32x2*>(src + u * 8);
            const int e = scale(t, 0);
#pragma unroll
            for (int j = 0; j < 8; ++j) rows[t * ST + e0 + j] = value_bits<T>(__builtin_amdgcn_ldexpf(code_at(w, j), e));
          } else {
            const int ln = u & 63, half = (u >> 6) & 1, st = u >> 7, t = half * 16 + (ln & 15), e0 = st * 32 + 8 * (ln >> 4);
            const u32x4 w = *reinterpret_cast<const u32x4*>(src + u * 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) *reinterpret_cast<uint32_t*>(rows + t * ST + e0 + 2 * j) = w[j];
          }
        }
      } else {
        const char* src = static_cast<const char*>(c.v) + paged_block_off(c, b.page, hk, b.blk, c.v_head, VT * 512) * (Q8 ? 1 : 2);
        for (int u = threadIdx.x; u < VT * 64; u += kThreads) {
          if constexpr (Q8) {
            const int ln = (u >> 1) & 63, d = ((u >> 7) * 2 + (u & 1)) * 16 + (ln & 15), t0 = 4 * (ln >> 4);
            const u32x2 w = *reinterpret_cast<const u32x2*>(src + u * 8);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int t = t0 + 16 * (j >> 2) + (j & 3);
              rows[t * ST + d] = value_bits<T>(__builtin_amdgcn_ldexpf(code_at(w, j), scale(t, 1)));
            }
          } else {
            const int ln = u & 63, d = (u >> 6) * 16 + (ln & 15), t0 = 4 * (ln >> 4);
            const u32x4 w = *reinterpret_cast<const u32x4*>(src + u * 16);
#pragma unroll
            for (int j = 0; j < 8; ++j) rows[(t0 + 16 * (j >> 2) + (j & 3)) * ST + d] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
          }
        }
      }
    }
    __syncthreads();
    for (int t = wave; t < kBlockKeys; t += kThreads / 64) {
      if (!live(t)) continue;
      const int64_t n = b.seg.row0 + b.i0 + t;
      if (!which) {
        uint16_t* dst = static_cast<uint16_t*>(p.k) + b.seg.batch * p.k_s[0] + hk * p.k_s[1] + n * p.k_s[2];
        for (int x = lane; x < E; x += 64) {
          const int e = x >= 2 * R ? x : (x & 1) * R + (x >> 1);
          dst[x] = b.page >= 0 ? rows[t * ST + e] : (uint16_t)0;
        }
      } else {
        uint16_t* dst = static_cast<uint16_t*>(p.v) + b.seg.batch * p.v_s[0] + hk * p.v_s[1] + n * p.v_s[2];
        for (int x = lane; x < D; x += 64) dst[x] = b.page >= 0 ? rows[t * ST + x] : (uint16_t)0;
      }
    }
  }
}

template <typename T, bool Q8, int VT>
hipError_t run_rows(const PagedRowsParams& p, bool write, hipStream_t s) {
  const dim3 grid((unsigned)p.blocks, p.c.Hk);
  return write ? launch_named("paged_write", paged_write_kernel<T, Q8, VT>, grid, dim3(kThreads), s, p)
               : launch_named("paged_read", paged_read_kernel<T, Q8, VT>, grid, dim3(kThreads), s, p);
}

template <typename T, bool Q8>
hipError_t run_rows_tiles(const PagedRowsParams& p, bool write, hipStream_t s) {
  switch (p.c.tiles) {
    case 2: return run_rows<T, Q8, 2>(p, write, s);
    case 4: return run_rows<T, Q8, 4>(p, write, s);
    case 6: return run_rows<T, Q8, 6>(p, write, s);
    case 8: return run_rows<T, Q8, 8>(p, write, s);
    case 16: return run_rows<T, Q8, 16>(p, write, s);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_rows(const PagedRowsParams& p, bool write, int dtype, bool q8, hipStream_t s) {
  if (dtype == 2) return q8 ? run_rows_tiles<BF16, true>(p, write, s) : run_rows_tiles<BF16, false>(p, write, s);
  return q8 ? run_rows_tiles<F16, true>(p, write, s) : run_rows_tiles<F16, false>(p, write, s);
}

}  // namespace

hipError_t launch_paged_write(const PagedRowsParams& p, int dtype, bool q8, hipStream_t s) { return launch_rows(p, true, dtype, q8, s); }
hipError_t launch_paged_read(const PagedRowsParams& p, int dtype, bool q8, hipStream_t s) { return launch_rows(p, false, dtype, q8, s); }

}  // namespace pope
