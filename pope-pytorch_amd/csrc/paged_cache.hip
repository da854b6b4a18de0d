// Rows into the paged cache and out of it (gfx950).
//
//   write  K_hat = [softplus(k) cos t, softplus(k) sin t, k], t = F + bias, rounded once: to 16 bits, or to e4m3 codes
//          x 2^-e with one e per (token, head): the smallest with max |x| <= 448 2^e.  A power of two scales exactly, so
//          codes of 16-bit values depend on no rounding but e4m3's own.
//   read   the rows back, K_hat with (cos, sin) pairs interleaved as apply_pope_to_qk lays them out.
//
// A workgroup has the block of 32 slots of one head that a 16-bit MFMA operand spans (paged_index.hpp): rows cross LDS
// between the callers' row order and the pages' operand order, so both sides of the copy are contiguous.  A thread has eight
// columns of a row (16-byte loads, all of a workgroup's in flight at once).  Slots of other tokens in the block are not
// touched: units of 16 bytes are stored whole only where all their tokens are written.
//
// Reads are bound by HBM, and by the launch where there is little to move: 8 x 8,192 tokens x 16 heads, D 64, R 64, 805 MB in
// 149 us (5.4 TB/s; a copy reaches 4.7, half of it writes); 8 x 500 x 8, D 72, R 40, 8 bits, 18 MB in 8 us.  Writes of many
// tokens are not, by half: 4 x 2,048 tokens x 8 heads, D 128, R 64, to 8 bits, 57 MB in 25 us (2.3 TB/s); 2,047 x 8, D 256,
// R 256, fp16, 44 MB in 23.5 us (1.9 TB/s).  Every head computes the sines and cosines of its F + bias (with softplus about 100
// vector instructions per rotated column), and load, transform and store stand in turn between barriers, in about one
// round of workgroups.  One token of 16 sequences: 4 us.
//
// The angle F + bias is kept as a sum of two floats (in one, at position 32,768, it would be off by up to 2e-3 rad) and the
// functions are accurate to about an ulp, so that a stored value is the rounding of the exact one except next to a rounding
// border.
#include <type_traits>

#include "paged_dev.hpp"

namespace pope {

namespace {

constexpr int kThreads = 256;

// sin and cos of a + b: the sum as hi + lo (exact), reduced by multiples of pi / 2 (Cody and Waite: pi / 2 in parts whose
// products with the multiple leave no error above 2^-24; in fp64 from 2^20 on, where the multiple outgrows them), then
// Taylor's series on |r| <= pi / 4 (the first terms left out are below 2e-9 and 4e-10).
__device__ __forceinline__ void sincos_sum(float a, float b, float* s, float* c) {
#pragma clang fp contract(off)
  constexpr double kHalfPi = 1.57079632679489661923;
  constexpr float p1 = (float)kHalfPi, p2 = (float)(kHalfPi - (double)p1);
  const float hi = a + b, bb = hi - a, lo = (a - (hi - bb)) + (b - bb);
  float k = __builtin_rintf(hi * 0.63661977236758134308f);
  float r = fmaf(-k, p2, fmaf(-k, p1, hi)) + lo;
  int quarter = (int)k & 3;
  if (fabsf(hi) >= 1048576.f) {
    POPE_COLD_PATH();
    const double t = (double)a + (double)b, q = __builtin_rint(t / kHalfPi);
    r = (float)__builtin_fma(-q, kHalfPi, t);
    quarter = (int)(long long)q & 3;
  }
  const float z = r * r;
  const float sr = fmaf(r * z, fmaf(z, fmaf(z, fmaf(z, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), r);
  const float cr = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.f / 3628800, 1.f / 40320), -1.f / 720), 1.f / 24), -0.5f), 1.f);
  const float u = quarter & 1 ? cr : sr, v = quarter & 1 ? sr : cr;
  *s = quarter & 2 ? -u : u;
  *c = (quarter + 1) & 2 ? -v : v;
}

// softplus to about an ulp: max(x, 0) + log(1 + e), e = e^-|x|: the exponent's product in two parts, and the logarithm as
// 2 artanh(y), y = e / (2 + e) <= 1/3 (the series' first term left out is below 1e-9).  An e below 2^-126 (x < -87.3) is 0.
__device__ __forceinline__ float softplus_accurate(float x) {
  constexpr double kL2e = 1.44269504088896340736;
  constexpr float l1 = (float)kL2e, l2 = (float)(kL2e - (double)l1);
  const float n = -fabsf(x), t = n * l1, rest = fmaf(n, l1, -t) + n * l2;
  const float e0 = __builtin_amdgcn_exp2f(t), e = fmaf(e0, rest * kLn2, e0);
  const float den = 2.f + e, q0 = __builtin_amdgcn_rcpf(den), q = fmaf(q0, fmaf(-den, q0, 1.f), q0);
  const float y0 = e * q, y = fmaf(q, fmaf(-y0, den, e), y0), z = y * y;
  const float g = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, 1.f / 17, 1.f / 15), 1.f / 13), 1.f / 11), 1.f / 9), 1.f / 7), 1.f / 5), 1.f / 3);
  const float r = fmaf(2.f * y * z, g, 2.f * y);
  return fabsf(x) < 104.f ? fmaxf(x, 0.f) + r : x < 0.f ? 0.f : x;   // beyond: e = 0; NaN stays NaN
}

// Biased exponent of the row's power of two.
__device__ __forceinline__ int row_exponent(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, -126), 126) + 127;
}

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

// Eight elements of a row from column d0 on (zeros past `cols`).
__device__ __forceinline__ u32x4 load_row8(const uint16_t* src, int d0, int cols, bool vec) {
  u32x4 w = {0, 0, 0, 0};
  if (vec) {
    w = *reinterpret_cast<const u32x4*>(src + d0);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (d0 + k < cols) w[k >> 1] |= (uint32_t)src[d0 + k] << (16 * (k & 1));
  }
  return w;
}

template <typename T, bool Q8, int VT>
__global__ __launch_bounds__(kThreads) void paged_write_kernel(PagedRowsParams p) {
  // rows in LDS, 16-bit elements or codes: K_hat (at most 2 D columns) and V, strides an odd number of 16-byte units
  typedef std::conditional_t<Q8, uint8_t, uint16_t> Held;
  constexpr int kPad = Q8 ? 16 : 8, KST = VT * 32 + kPad, VST = VT * 16 + kPad;
  constexpr int kTurns = (kBlockKeys * VT * 2 + kThreads - 1) / kThreads;   // chunks of eight columns per thread
  __shared__ __attribute__((aligned(16))) Held krows[kBlockKeys * KST];
  __shared__ __attribute__((aligned(16))) Held vrows[kBlockKeys * VST];
  __shared__ uint32_t amax[2][kBlockKeys];   // largest finite magnitude of a row, as the bits of a float
  const PagedCache& c = p.c;
  const int hk = blockIdx.y, tid = threadIdx.x;
  const Block b = find_block(c, blockIdx.x);
  if (!b.any || b.page < 0) return;
  // slots t of the block that the call writes
  auto live = [&](int t) { return (unsigned)(b.i0 + t) < (unsigned)b.seg.n; };
  const int D = c.D, R = c.R, KE = c.steps * 32;
  const bool whole = R % 8 == 0;

  // A thread's chunks: four side by side in a row, 32 rows, then the next four: a wave's are all rotated or mostly not, and a
  // chunk's sine, cosine and softplus are most of the work (rows' chunks side by side: both branches in every wave).
  u32x4 kin[kTurns], vin[kTurns];
  f32x4 fin[kTurns][2], bin[kTurns][2];
#pragma unroll
  for (int u = 0; u < kTurns; ++u) {
    const int t = (tid >> 2) % kBlockKeys, d0 = ((tid & 3) + 4 * (tid / 128 + 2 * u)) * 8;
    kin[u] = vin[u] = u32x4{0, 0, 0, 0};
    fin[u][0] = fin[u][1] = bin[u][0] = bin[u][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (!live(t) || d0 >= D) continue;
    const int64_t n = b.seg.row0 + b.i0 + t;
    kin[u] = load_row8(static_cast<const uint16_t*>(p.k) + b.seg.batch * p.k_s[0] + hk * p.k_s[1] + n * p.k_s[2], d0, D, p.k_vec);
    vin[u] = load_row8(static_cast<const uint16_t*>(p.v) + b.seg.batch * p.v_s[0] + hk * p.v_s[1] + n * p.v_s[2], d0, D, p.v_vec);
    if (d0 < R) {
      const float* f = p.freqs + b.seg.batch * p.f_s[0] + n * p.f_s[1] + d0;
      const float* bias = p.bias + hk * p.bias_sh + d0;
      if (p.f_vec) {   // R a multiple of 8, rows of angles and bias 16-byte aligned
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          fin[u][k] = *reinterpret_cast<const f32x4*>(f + 4 * k);
          bin[u][k] = *reinterpret_cast<const f32x4*>(bias + 4 * k);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (d0 + k < R) {
            fin[u][k >> 2][k & 3] = f[k];
            bin[u][k >> 2][k & 3] = bias[k];
          }
      }
    }
  }
  if (Q8 && tid < 2 * kBlockKeys) amax[tid / kBlockKeys][tid % kBlockKeys] = 0;
  // what a row has behind its columns: zeros (keys; value columns past D are read by nothing but whole tiles)
  for (int it = tid; it < kBlockKeys * (KE - D - R); it += kThreads) krows[it % kBlockKeys * KST + D + R + it / kBlockKeys] = 0;
  if (D < VT * 16)
    for (int it = tid; it < kBlockKeys * (VT * 16 - D); it += kThreads) vrows[it % kBlockKeys * VST + D + it / kBlockKeys] = 0;
  __syncthreads();

  float ka[kTurns][8], kb[kTurns][8];   // cosine part or raw value, sine part
#pragma unroll
  for (int u = 0; u < kTurns; ++u) {
    const int t = (tid >> 2) % kBlockKeys, d0 = ((tid & 3) + 4 * (tid / 128 + 2 * u)) * 8;
    unpack8<T>(kin[u], ka[u]);
    if (d0 < R) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float sn, cs;
        sincos_sum(fin[u][k >> 2][k & 3], bin[u][k >> 2][k & 3], &sn, &cs);
        const float m = softplus_accurate(ka[u][k]);
        const bool rot = d0 + k < R;
        kb[u][k] = rot ? m * sn : 0.f;
        ka[u][k] = rot ? m * cs : ka[u][k];
      }
    }
    if (Q8 && live(t) && d0 < D) {
      float mk = 0.f, mv = 0.f, v[8];
      unpack8<T>(vin[u], v);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (finite_f(ka[u][k])) mk = fmaxf(mk, fabsf(ka[u][k]));
        if (d0 < R && finite_f(kb[u][k])) mk = fmaxf(mk, fabsf(kb[u][k]));
        if (finite_f(v[k])) mv = fmaxf(mv, fabsf(v[k]));
      }
      atomicMax(&amax[0][t], __float_as_uint(mk));
      atomicMax(&amax[1][t], __float_as_uint(mv));
    }
  }
  if constexpr (Q8) {
    __syncthreads();
    if (tid < 2 * kBlockKeys) {
      const int which = tid / kBlockKeys, t = tid % kBlockKeys;
      if (live(t))
        c.scales[paged_scale_base(c, b.page, hk, b.blk) + paged_scale_off(t, which)] = (uint8_t)row_exponent(__uint_as_float(amax[which][t]));
    }
  }
#pragma unroll
  for (int u = 0; u < kTurns; ++u) {
    const int t = (tid >> 2) % kBlockKeys, d0 = ((tid & 3) + 4 * (tid / 128 + 2 * u)) * 8;
    if (d0 >= D) continue;
    float v[8];
    unpack8<T>(vin[u], v);
    // eight columns from e on, whole or one by one
    auto put = [&](Held* row, int e, const float* x, int which, bool vec, int count) {
      if constexpr (Q8) {
        const float inv = __uint_as_float((uint32_t)(254 - row_exponent(__uint_as_float(amax[which][t]))) << 23);
        auto code = [&](int k) {   // x 2^-e, NaN where x is not finite
          const float y = x[k] * inv;
          return finite_f(y) ? y : __builtin_nanf("");
        };
        u32x2 w;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(code(4 * k), code(4 * k + 1), 0, false);
          w[k] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(code(4 * k + 2), code(4 * k + 3), lo, true);
        }
        if (vec) {
          *reinterpret_cast<u32x2*>(row + e) = w;
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (k < count) row[e + k] = (uint8_t)(w[k >> 2] >> (8 * (k & 3)));
        }
      } else {
        if (vec) {
          *reinterpret_cast<u32x4*>(row + e) = u32x4{T::pack2(x[0], x[1]), T::pack2(x[2], x[3]), T::pack2(x[4], x[5]), T::pack2(x[6], x[7])};
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (k < count) row[e + k] = T::bits(x[k]);
        }
      }
    };
    Held* row = krows + t * KST;
    const bool full = d0 + 8 <= D;
    if (d0 >= R) {
      put(row, R + d0, ka[u], 0, whole && full, D - d0);
    } else {
      const int rot = R - d0;   // rotated columns of the chunk, if fewer than 8
      put(row, d0, ka[u], 0, rot >= 8, rot);
      put(row, R + d0, kb[u], 0, whole, rot);
      if (rot < 8) {            // the others stand R columns further on
        float y[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) y[k] = ka[u][k];
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k >= rot && d0 + k < D) {
            const float one[8] = {y[k], 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            put(row, R + d0 + k, one, 0, false, 1);
          }
      }
    }
    if (!Q8 && full) *reinterpret_cast<u32x4*>(vrows + t * VST + d0) = vin[u];
    else put(vrows + t * VST, d0, v, 1, full, D - d0);
  }
  __syncthreads();

  // ---- units of 16 bytes (8-bit: 8) into the block, in operand order ------------------------------------------
  Held* kdst = static_cast<Held*>(c.k) + paged_block_off(c, b.page, hk, b.blk, c.k_head, KE * 32);
  Held* vdst = static_cast<Held*>(c.v) + paged_block_off(c, b.page, hk, b.blk, c.v_head, VT * 512);
  typedef std::conditional_t<Q8, u32x2, u32x4> Unit;
  for (int u = tid; u < c.steps * 128; u += kThreads) {   // 16-bit: (step, half, lane); 8-bit: (step, lane, half)
    const int half = Q8 ? u & 1 : (u >> 6) & 1, ln = Q8 ? (u >> 1) & 63 : u & 63, t = half * 16 + (ln & 15), e0 = (u >> 7) * 32 + 8 * (ln >> 4);
    if (live(t)) *reinterpret_cast<Unit*>(kdst + u * 8) = *reinterpret_cast<const Unit*>(krows + t * KST + e0);
  }
  for (int u = tid; u < VT * 64; u += kThreads) {   // 16-bit: (tile, lane); 8-bit: (tile pair, lane, tile of the pair)
    const int ln = Q8 ? (u >> 1) & 63 : u & 63, d = (Q8 ? (u >> 7) * 2 + (u & 1) : u >> 6) * 16 + (ln & 15), t0 = 4 * (ln >> 4);
    Held w[8];
    bool all = true;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int t = t0 + 16 * (j >> 2) + (j & 3);
      all = all && live(t);
      w[j] = vrows[t * VST + d];
    }
    if (all) {
      Unit x;
#pragma unroll
      for (int k = 0; k < (Q8 ? 2 : 4); ++k)
        x[k] = Q8 ? w[(4 * k) & 7] | ((uint32_t)w[(4 * k + 1) & 7] << 8) | ((uint32_t)w[(4 * k + 2) & 7] << 16) | ((uint32_t)w[(4 * k + 3) & 7] << 24)
                  : w[2 * k] | ((uint32_t)w[2 * k + 1] << 16);
      *reinterpret_cast<Unit*>(vdst + u * 8) = x;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (live(t0 + 16 * (j >> 2) + (j & 3))) vdst[u * 8 + j] = w[j];
    }
  }
}

// 8-bit rows: the code of a row's largest may stand for more than the 16-bit type holds (fp16: 65536, bf16: 2^128), where the
// row's exponent is above kMostExp (448 2^kMostExp is in range).  e4m3 has no infinity, so that an infinity of a dequantised
// pair of values is such a code, and becomes the type's largest.
template <typename T>
constexpr int kMostExp = T::kCode == 1 ? 7 : 119;
template <typename T>
__device__ __forceinline__ uint32_t in_range(uint32_t pair) {
  constexpr uint32_t kInf = T::kCode == 1 ? 0x7c007c00u : 0x7f807f80u;
  const uint32_t other = (((pair ^ kInf) & 0x7fff7fffu) + 0x7fff7fffu) & 0x80008000u;
  return pair - ((other ^ 0x80008000u) >> 15);
}

template <typename T, bool Q8, int VT>
__global__ __launch_bounds__(kThreads) void paged_read_kernel(PagedRowsParams p) {
  constexpr int ST = VT * 32 + 8;   // an odd number of 16-byte units
  __shared__ __attribute__((aligned(16))) uint16_t rows[kBlockKeys * ST];
  const PagedCache& c = p.c;
  const int hk = blockIdx.y, lane = threadIdx.x & 63, wave = wave_id();
  const Block b = find_block(c, blockIdx.x);
  if (!b.any) return;
  auto live = [&](int t) { return (unsigned)(b.i0 + t) < (unsigned)b.seg.n; };
  const uint8_t* scales = Q8 && b.page >= 0 ? c.scales + paged_scale_base(c, b.page, hk, b.blk) : nullptr;
  const int D = c.D, R = c.R, E = D + R, KE = c.steps * 32;
  auto scale = [&](int t, int which) { return (int)scales[paged_scale_off(t, which)] - 127; };
  const bool wide = Q8 && scales && __any((int)scales[lane] - 127 > kMostExp<T>);   // of the block's rows, some may leave the type
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
            for (int j = 0; j < 8; j += 2)
              *reinterpret_cast<uint32_t*>(rows + t * ST + e0 + j) = T::pack2(__builtin_amdgcn_ldexpf(code_at(w, j), e), __builtin_amdgcn_ldexpf(code_at(w, j + 1), e));
          } else {
            const int ln = u & 63, half = (u >> 6) & 1, st = u >> 7, t = half * 16 + (ln & 15), e0 = st * 32 + 8 * (ln >> 4);
            *reinterpret_cast<u32x4*>(rows + t * ST + e0) = *reinterpret_cast<const u32x4*>(src + u * 16);
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
              rows[t * ST + d] = T::bits(__builtin_amdgcn_ldexpf(code_at(w, j), scale(t, 1)));
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
    const int cols = which ? D : E;
    if (which ? p.v_vec : p.k_vec && R % 4 == 0) {   // 16 bytes at a time: eight columns, or four (cos, sin) pairs
      for (int u = threadIdx.x; u < kBlockKeys * (VT * (which ? 2 : 4)); u += kThreads) {
        const int t = u / (VT * (which ? 2 : 4)), x = u % (VT * (which ? 2 : 4)) * 8;
        if (!live(t) || x >= cols) continue;
        const int64_t n = b.seg.row0 + b.i0 + t;
        const uint16_t* row = rows + t * ST;
        u32x4 w = {0, 0, 0, 0};
        if (b.page >= 0) {
          if (which || x >= 2 * R) {
            w = *reinterpret_cast<const u32x4*>(row + x);
          } else {
            const u32x2 cs = *reinterpret_cast<const u32x2*>(row + x / 2), sn = *reinterpret_cast<const u32x2*>(row + R + x / 2);
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = ((cs[k >> 1] >> (16 * (k & 1))) & 0xffffu) | (sn[k >> 1] >> (16 * (k & 1))) << 16;
          }
        }
        if (Q8 && wide) {
          POPE_COLD_PATH();
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = in_range<T>(w[k]);
        }
        uint16_t* dst = which ? static_cast<uint16_t*>(p.v) + b.seg.batch * p.v_s[0] + hk * p.v_s[1] + n * p.v_s[2]
                              : static_cast<uint16_t*>(p.k) + b.seg.batch * p.k_s[0] + hk * p.k_s[1] + n * p.k_s[2];
        *reinterpret_cast<u32x4*>(dst + x) = w;
      }
    } else {
      for (int t = wave; t < kBlockKeys; t += kThreads / 64) {
        if (!live(t)) continue;
        const int64_t n = b.seg.row0 + b.i0 + t;
        uint16_t* dst = which ? static_cast<uint16_t*>(p.v) + b.seg.batch * p.v_s[0] + hk * p.v_s[1] + n * p.v_s[2]
                              : static_cast<uint16_t*>(p.k) + b.seg.batch * p.k_s[0] + hk * p.k_s[1] + n * p.k_s[2];
        for (int x = lane; x < cols; x += 64) {
          const int e = which || x >= 2 * R ? x : (x & 1) * R + (x >> 1);
          const uint16_t w = b.page >= 0 ? rows[t * ST + e] : (uint16_t)0;
          dst[x] = Q8 && wide ? (uint16_t)in_range<T>(w) : w;
        }
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
