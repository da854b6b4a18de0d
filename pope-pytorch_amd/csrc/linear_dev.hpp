// Device helpers of the linear attention's kernels: segments of sequences, and rows on their way into LDS.
#pragma once
#include "linear.hpp"
#include "pope_common.hpp"

namespace pope {

typedef __attribute__((ext_vector_type(2))) float f32x2;
constexpr float kF32Max = 3.402823466e38f, kBf16Max = 3.3895313892515355e38f;

// The norm of a row whose squares pass fp32's range is that of the row times 2^-100: its largest value, 2^59 at least (of up to 512),
// is between 2^-41 and 2^28 then, and the eps that goes with it, times 2^-200, nothing beside that.
constexpr float kNormDown = 0x1p-100f;

// ---------------------------------------------------------------- segments

struct LinSeg {
  int seq, batch;   // seq < 0: none
  int row0, len;    // rows row0 .. row0 + len - 1 of the batch entry
  int m;            // which of the sequence's; where there is none: how many segments there are
};
constexpr int kLinNone = 0x7fffffff;   // behind every segment

__device__ __forceinline__ int lin_bound(const LinSeqs& q, int i) { return min(max(q.cu[i], 0), q.N); }

// Segments of the packed sequences before `seq` (all lanes of a wave call it), and of itself.
__device__ __forceinline__ int lin_first(const LinSeqs& q, int seq, int* row0, int* rows) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int s0 = 0; s0 < seq; s0 += 64) {
    const int s = s0 + lane;
    int c = s < seq ? (max(lin_bound(q, s + 1) - lin_bound(q, s), 0) + q.L - 1) / q.L : 0;
#pragma unroll
    for (int i = 1; i < 64; i *= 2) c += __shfl_xor(c, i, 64);
    before += c;
  }
  *row0 = lin_bound(q, seq);
  *rows = max(lin_bound(q, seq + 1) - *row0, 0);
  return __builtin_amdgcn_readfirstlane(before);
}

// Segment `at` of the call (uniform; all lanes of a wave call it).
__device__ __forceinline__ LinSeg lin_segment(const LinSeqs& q, int at) {
  LinSeg g;
  if (!q.cu) {
    g.seq = g.batch = at / q.M;
    g.m = at - g.seq * q.M;
    g.row0 = g.m * q.L;
    g.len = min(q.L, q.N - g.row0);
    return g;
  }
  const int lane = threadIdx.x & 63;
  g.seq = -1;
  g.batch = 0;
  g.row0 = g.len = g.m = 0;
  int before = 0;
  for (int s0 = 0; s0 < q.B; s0 += 64) {
    const int s = s0 + lane;
    int a = 0, n = 0;
    if (s < q.B) a = lin_bound(q, s), n = max(lin_bound(q, s + 1) - a, 0);
    const int own = (n + q.L - 1) / q.L;
    int upto = own;
#pragma unroll
    for (int i = 1; i < 64; i *= 2) {
      const int x = __shfl_up(upto, i, 64);
      upto += lane >= i ? x : 0;
    }
    const uint64_t above = __ballot(before + upto > at);
    if (above) {
      const int i = __builtin_ctzll(above);
      const int first = before + __builtin_amdgcn_readlane(upto - own, i);
      g.seq = s0 + i;
      g.m = at - first;
      g.row0 = __builtin_amdgcn_readlane(a, i) + g.m * q.L;
      g.len = min(q.L, __builtin_amdgcn_readlane(n, i) - g.m * q.L);
      return g;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  g.m = before;
  return g;
}

// ---------------------------------------------------------------- decay

// g^n from log2 g.  g^0 is 1 whatever g is (a decay of 0 has log2 g = -inf).
__device__ __forceinline__ float lin_power(float lg, int n) { return n == 0 ? 1.f : __builtin_amdgcn_exp2f(lg * (float)n); }
__device__ __forceinline__ float lin_log2(const LinCall& c, int hk) { return c.log_decay ? c.log_decay[hk] * kLog2e : 0.f; }

// ---------------------------------------------------------------- rows

// sin and cos of x + 2 pi turns: as sincos_rev, with `turns` in [-1/2, 1/2] added to the fraction, so that the sum of a far
// position's angle and a bias is not rounded.
__device__ __forceinline__ void sincos_turns(float x, float turns, float* s, float* c) {
#pragma clang fp contract(off)
  constexpr float kHi = 0.15915494f;
  constexpr float kLo = (float)(0.15915494309189533577 - (double)0.15915494f);
  const float hi = x * kHi;
  const float lo = fmaf(x, kHi, -hi) + x * kLo;
  const float fr = (hi - __builtin_rintf(hi)) + (lo + turns);
  *s = __builtin_amdgcn_sinf(fr);
  *c = __builtin_amdgcn_cosf(fr);
}
// A bias as turns.
__device__ __forceinline__ float lin_turns(float b) {
  const float t = b * 0.15915494309189533577f;
  return t - __builtin_rintf(t);
}

// How a kernel takes its rows: kOne, bf16 rows as operands of one part; kTwo, rows of any type as the sum of two bf16 parts
// (exactly, for 16-bit rows; 2^-16 off for fp32 ones).
enum LinParts { kOne = 1, kTwo = 2 };

// Rows near each other are addressed by a base that a wave shares and a 32-bit offset in bytes (a chunk of 64 rows, row strides below
// 2^22 elements): one register a load, the same in every chunk.
__device__ __forceinline__ char* lin_uniform(const void* p) {
  const uint64_t x = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x), hi = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32));
  return (char*)(__attribute__((address_space(1))) char*)((uint64_t)hi << 32 | lo);   // global memory: else loads would ask LDS too
}
// Base of row `row` of a (batch, head).
__device__ __forceinline__ char* lin_base(const LinRows& r, int batch, int h, int64_t row) {
  return lin_uniform(static_cast<char*>(r.p) + (batch * r.s[0] + h * r.s[1] + row * r.s[2]) * lin_size(r.type));
}

// Eight elements of a row, as they are in memory.
template <int PL>
struct LinRaw {
  u32x4 a;
};
template <>
struct LinRaw<kTwo> {
  u32x4 a, b;   // b: of fp32 rows
};
// softplus and its derivative, of one exponential.
__device__ __forceinline__ void lin_soft(float x, float* soft, float* slope) {
  const float e = __builtin_amdgcn_exp2f(-fabsf(x) * kLog2e), r = __builtin_amdgcn_rcpf(1.f + e);
  *soft = fmaf(__builtin_amdgcn_logf(1.f + e), kLn2, fmaxf(x, 0.f));
  *slope = x >= 0.f ? r : e * r;
}

// base + off: the row.  whole: r.vec, known before.
template <int PL>
__device__ __forceinline__ LinRaw<PL> lin_load8(const LinRows& r, const char* base, uint32_t off, int d0, bool whole) {
  LinRaw<PL> w{};
  if constexpr (PL == kTwo) {
    if (whole) {   // both loads, one of them twice for 16-bit rows: no branch
      off += d0 * lin_size(r.type);
      w.a = *reinterpret_cast<const u32x4*>(base + off);
      w.b = *reinterpret_cast<const u32x4*>(base + (off + (r.type == 0 ? 16 : 0)));
      return w;
    }
    if (r.type == 0) {
      const uint32_t* p = reinterpret_cast<const uint32_t*>(base + (off + 4 * d0));
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (d0 + k < r.cols) w.a[k] = p[k];
        if (d0 + 4 + k < r.cols) w.b[k] = p[4 + k];
      }
      return w;
    }
  }
  off += 2 * d0;
  if (whole) {
    w.a = *reinterpret_cast<const u32x4*>(base + off);
  } else {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(base + off);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (d0 + k < r.cols) w.a[k >> 1] |= (uint32_t)p[k] << (16 * (k & 1));
  }
  return w;
}
template <int PL>   // `at`: elements before the row
__device__ __forceinline__ LinRaw<PL> lin_load8(const LinRows& r, int64_t at, int d0) {
  return lin_load8<PL>(r, static_cast<const char*>(r.p) + at * (PL == kTwo ? lin_size(r.type) : 2), 0u, d0, r.vec);
}
template <int PL>
__device__ __forceinline__ void lin_unpack8(const LinRaw<PL>& w, int type, float* f) {
  if constexpr (PL == kTwo) {
    if (type == 0) {
#pragma unroll
      for (int k = 0; k < 4; ++k) f[k] = __uint_as_float(w.a[k]), f[4 + k] = __uint_as_float(w.b[k]);
      return;
    }
    if (type == 1) return unpack8<F16>(w.a, f);
  }
  unpack8<BF16>(w.a, f);
}
// An fp32 value of rows that become bf16 parts: finite ones above the largest bf16 (by 2^-8 of it at most) count as that.  Their first
// part would round to infinity, and 0 x infinity of a row behind would be NaN.
__device__ __forceinline__ float lin_part(uint32_t w) {
  const float v = __uint_as_float(w);
  return fabsf(v) <= kF32Max ? __builtin_amdgcn_fmed3f(v, -kBf16Max, kBf16Max) : v;
}
template <int PL>
__device__ __forceinline__ void lin_row8(const LinRaw<PL>& w, int type, float* f) {
  if constexpr (PL == kTwo) {
    if (type == 0) {
#pragma unroll
      for (int k = 0; k < 4; ++k) f[k] = lin_part(w.a[k]), f[4 + k] = lin_part(w.b[k]);
      return;
    }
  }
  lin_unpack8<PL>(w, type, f);
}
// One element.
template <int PL>
__device__ __forceinline__ float lin_get(const LinRows& r, int64_t at) {
  if constexpr (PL == kTwo) {
    if (r.type == 0) return static_cast<const float*>(r.p)[at];
    if (r.type == 1) return F16::to_float(static_cast<const uint16_t*>(r.p)[at]);
  }
  return BF16::to_float(static_cast<const uint16_t*>(r.p)[at]);
}
template <int PL>
__device__ __forceinline__ void lin_set(const LinRows& r, int64_t at, float v) {
  if constexpr (PL == kTwo) {
    if (r.type == 0) {
      static_cast<float*>(r.p)[at] = v;
      return;
    }
    if (r.type == 1) {
      static_cast<uint16_t*>(r.p)[at] = F16::bits(v);
      return;
    }
  }
  static_cast<uint16_t*>(r.p)[at] = BF16::bits(v);
}
template <int PL>
__device__ __forceinline__ void lin_put_value(const LinRows& r, char* base, uint32_t off, int d, float v) {
  if constexpr (PL == kTwo) {
    if (r.type == 0) {
      *reinterpret_cast<float*>(base + (off + 4 * d)) = v;
      return;
    }
    if (r.type == 1) {
      *reinterpret_cast<uint16_t*>(base + (off + 2 * d)) = F16::bits(v);
      return;
    }
  }
  *reinterpret_cast<uint16_t*>(base + (off + 2 * d)) = BF16::bits(v);
}
// Four elements of an output row from column d on (r.vec: d a multiple of 4, whole units).
template <int PL>
__device__ __forceinline__ void lin_set4(const LinRows& r, char* base, uint32_t off, int d, f32x4 v) {
  if (d >= r.cols) return;
  if (!r.vec) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (d + k < r.cols) lin_put_value<PL>(r, base, off, d + k, v[k]);
    return;
  }
  if constexpr (PL == kTwo) {
    if (r.type == 0) {
      *reinterpret_cast<f32x4*>(base + (off + 4 * d)) = v;
      return;
    }
    if (r.type == 1) {
      *reinterpret_cast<u32x2*>(base + (off + 2 * d)) = u32x2{F16::pack2(v[0], v[1]), F16::pack2(v[2], v[3])};
      return;
    }
  }
  *reinterpret_cast<u32x2*>(base + (off + 2 * d)) = u32x2{BF16::pack2(v[0], v[1]), BF16::pack2(v[2], v[3])};
}
// Two elements at an even place of an aligned row, as they are in memory.
template <int PL>
struct LinPair { uint32_t w; };
template <>
struct LinPair<kTwo> { uint32_t w, v; };   // v: the second of fp32 rows
template <int PL>
__device__ __forceinline__ LinPair<PL> lin_get2(const LinRows& r, const char* base, uint32_t off, int d) {
  LinPair<PL> o;
  off += d * lin_size(r.type);
  o.w = *reinterpret_cast<const uint32_t*>(base + off);
  if constexpr (PL == kTwo) o.v = *reinterpret_cast<const uint32_t*>(base + (off + (r.type == 0 ? 4 : 0)));
  return o;
}
template <int PL>
__device__ __forceinline__ float lin_get1(const LinRows& r, const char* base, uint32_t off, int d) {
  if constexpr (PL == kTwo) {
    if (r.type == 0) return lin_part(*reinterpret_cast<const uint32_t*>(base + (off + 4 * d)));
    if (r.type == 1) return F16::to_float(*reinterpret_cast<const uint16_t*>(base + (off + 2 * d)));
  }
  return BF16::to_float(*reinterpret_cast<const uint16_t*>(base + (off + 2 * d)));
}
template <int PL>
__device__ __forceinline__ void lin_unpack2(const LinPair<PL>& p, int type, float* v) {
  if constexpr (PL == kTwo) {
    if (type == 0) {
      v[0] = lin_part(p.w), v[1] = lin_part(p.v);
      return;
    }
    if (type == 1) {
      v[0] = F16::to_float((uint16_t)p.w), v[1] = F16::to_float((uint16_t)(p.w >> 16));
      return;
    }
  }
  v[0] = BF16::to_float((uint16_t)p.w), v[1] = BF16::to_float((uint16_t)(p.w >> 16));
}
template <int PL>
__device__ __forceinline__ void lin_set2(const LinRows& r, char* base, uint32_t off, int d, float a, float b) {
  if constexpr (PL == kTwo) {
    if (r.type == 0) {
      *reinterpret_cast<f32x2*>(base + (off + 4 * d)) = f32x2{a, b};
      return;
    }
    if (r.type == 1) {
      *reinterpret_cast<uint32_t*>(base + (off + 2 * d)) = F16::pack2(a, b);
      return;
    }
  }
  *reinterpret_cast<uint32_t*>(base + (off + 2 * d)) = BF16::pack2(a, b);
}
// Values of an array of one of the types.
__device__ __forceinline__ float lin_value(const void* p, int type, int64_t i) {
  return type == 0 ? static_cast<const float*>(p)[i] : type == 1 ? F16::to_float(static_cast<const uint16_t*>(p)[i]) : BF16::to_float(static_cast<const uint16_t*>(p)[i]);
}
__device__ __forceinline__ float lin_bias(const LinCall& c, int hk, int d) { return lin_value(c.bias, c.bias_type, hk * c.bias_sh + d); }

__device__ __forceinline__ void lin_angles8(const float* row, int d0, int R, bool vec, f32x4* f) {
  f[0] = f[1] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (d0 >= R) return;
  if (vec) {
    f[0] = *reinterpret_cast<const f32x4*>(row + d0);
    f[1] = *reinterpret_cast<const f32x4*>(row + d0 + 4);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (d0 + k < R) f[k >> 2][k & 3] = row[d0 + k];
  }
}

__device__ __forceinline__ const float* lin_angle_row(const LinCall& c, int batch, int row) {
  return c.freqs + (int64_t)batch * c.f_s[0] + (int64_t)row * c.f_s[1];
}

// A tile's place of column e in rows that the products read as operands of 32 columns, eight for each quarter of a wave:
// column 16 h + 4 q + i of a group of 32 at 8 q + 4 h + i, which is where a 16x16 result's rows (4 q + i of tile h) come back as an
// operand.  Only tiles read along their rows are laid out so; those read across them keep their columns.
template <bool PERM>
__device__ __forceinline__ int lin_place(int e) {
  return PERM ? (e & ~31) | ((e >> 2) & 3) << 3 | ((e >> 4) & 1) << 2 | (e & 3) : e;
}

// bf16 parts of fp32 values: one, rounded, or the sum of two (16 significant bits).
template <int PL>
__device__ __forceinline__ void lin_pack4(f32x4 v, u32x2* w) {
  w[0] = u32x2{BF16::pack2(v[0], v[1]), BF16::pack2(v[2], v[3])};
  if constexpr (PL == 2)
    w[1] = u32x2{BF16::pack2(v[0] - BF16::to_float((uint16_t)w[0][0]), v[1] - BF16::to_float((uint16_t)(w[0][0] >> 16))),
                 BF16::pack2(v[2] - BF16::to_float((uint16_t)w[0][1]), v[3] - BF16::to_float((uint16_t)(w[0][1] >> 16)))};
}

// A tile of rows in LDS: PL planes of `stride` elements a row, `plane` elements apart.
struct LinTile {
  uint16_t* p;
  int stride, plane;
};

// Eight columns from e on (e a multiple of 8), all inside the tile.
template <int PL, bool PERM>
__device__ __forceinline__ void lin_put8(const LinTile& t, int row, int e, const float* v) {
  u32x2 a[PL], b[PL];
  lin_pack4<PL>(f32x4{v[0], v[1], v[2], v[3]}, a);
  lin_pack4<PL>(f32x4{v[4], v[5], v[6], v[7]}, b);
#pragma unroll
  for (int l = 0; l < PL; ++l) {
    uint16_t* at = t.p + l * t.plane + row * t.stride;
    if constexpr (PERM) {
      *reinterpret_cast<u32x2*>(at + lin_place<true>(e)) = a[l];
      *reinterpret_cast<u32x2*>(at + lin_place<true>(e + 4)) = b[l];
    } else {
      *reinterpret_cast<u32x4*>(at + e) = u32x4{a[l][0], a[l][1], b[l][0], b[l][1]};
    }
  }
}
template <int PL, bool PERM>
__device__ __forceinline__ void lin_put1(const LinTile& t, int row, int e, float v) {
  const uint16_t h = BF16::bits(v);
  uint16_t* at = t.p + row * t.stride + lin_place<PERM>(e);
  *at = h;
  if constexpr (PL == 2) at[t.plane] = BF16::bits(v - BF16::to_float(h));
}

// Whether some of eight bf16 values is not finite.
__device__ __forceinline__ bool lin_odd8(u32x4 w) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) m |= (w[i] & 0x7fff7fffu) + 0x00800080u;   // carries into the sign where all exponent bits are set
  return (m & 0x80008000u) != 0;
}
// Eight columns of a tile from e on, as parts in registers.
template <int PL, bool PERM>
__device__ __forceinline__ void lin_put_parts(const LinTile& t, int row, int e, const u32x4* w) {
#pragma unroll
  for (int l = 0; l < PL; ++l) {
    uint16_t* at = t.p + l * t.plane + row * t.stride;
    if constexpr (PERM) {
      *reinterpret_cast<u32x2*>(at + lin_place<true>(e)) = u32x2{w[l][0], w[l][1]};
      *reinterpret_cast<u32x2*>(at + lin_place<true>(e + 4)) = u32x2{w[l][2], w[l][3]};
    } else {
      *reinterpret_cast<u32x4*>(at + e) = w[l];
    }
  }
}

// Eight columns of a plain row, from column e of the tile on.  Returns whether some value is not finite.
template <int PL, bool PERM>
__device__ __forceinline__ bool lin_put_plain(const LinTile& t, int row, int e, const LinRaw<PL>& x, int type) {
  if constexpr (PL == kOne) {
    lin_put_parts<1, PERM>(t, row, e, &x.a);
    return lin_odd8(x.a);
  } else {
    float v[8];
    lin_row8<PL>(x, type, v);
    bool odd = false;
#pragma unroll
    for (int k = 0; k < 8; ++k) odd = odd || !(fabsf(v[k]) <= kF32Max);
    lin_put8<PL, PERM>(t, row, e, v);
    return odd;
  }
}

// Eight columns d0 .. of a row, expanded: a the cosine part or the value, b the sine part of rotated dims; times `factor`.
// turns: the bias of the keys in LDS, or null.
template <int PL>
__device__ __forceinline__ void lin_polar8(const LinRaw<PL>& x8, int type, const f32x4* f, int d0, int R, float factor, const float* turns, float* a, float* b) {
  float x[8];
  lin_row8<PL>(x8, type, x);
  if (d0 < R) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float sn, cs;
      const bool rot = d0 + k < R;
      sincos_turns(f[k >> 2][k & 3], turns && rot ? turns[d0 + k] : 0.f, &sn, &cs);
      const float m = softplus_f(x[k]) * factor;
      a[k] = rot ? m * cs : x[k] * factor;
      b[k] = rot ? m * sn : 0.f;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) a[k] = x[k] * factor, b[k] = 0.f;
  }
}
// Their places in an expanded row: put8(e, eight values) where a chunk's columns start on a multiple of 8, else put1(e, value).
template <typename F8, typename F1>
__device__ __forceinline__ void lin_place8(int d0, int D, int R, const float* a, const float* b, F8&& put8, F1&& put1) {
  if (R % 8 == 0) {   // a chunk is all rotated or all not; columns behind the row (D no multiple of 8) are zeros
    if (d0 < R) {
      float w[16];
#pragma unroll
      for (int k = 0; k < 8; ++k) w[2 * k] = a[k], w[2 * k + 1] = b[k];
      put8(2 * d0, w);
      put8(2 * d0 + 8, w + 8);
    } else {
      put8(R + d0, a);
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int d = d0 + k;
    if (d >= D) break;
    put1(d < R ? 2 * d : R + d, a[k]);
    if (d < R) put1(2 * d + 1, b[k]);
  }
}

// Expanded rows to memory.
template <int PL>
__device__ __forceinline__ void lin_hat_put(const LinHat& t, int64_t row, int d0, int D, int R, const float* a, const float* b) {
  uint16_t* at = t.p + row * t.EP;
  lin_place8(d0, D, R, a, b,
             [&](int e, const float* v) {
               u32x2 lo[PL], hi[PL];
               lin_pack4<PL>(f32x4{v[0], v[1], v[2], v[3]}, lo);
               lin_pack4<PL>(f32x4{v[4], v[5], v[6], v[7]}, hi);
#pragma unroll
               for (int l = 0; l < PL; ++l) *reinterpret_cast<u32x4*>(at + l * t.plane + e) = u32x4{lo[l][0], lo[l][1], hi[l][0], hi[l][1]};
             },
             [&](int e, float v) {
               const uint16_t w = BF16::bits(v);
               at[e] = w;
               if constexpr (PL == 2) at[t.plane + e] = BF16::bits(v - BF16::to_float(w));
             });
}
// The zeros behind them, by THREADS threads.
template <int PL, int THREADS>
__device__ __forceinline__ void lin_hat_tail(const LinHat& t, int64_t row, int thread, int D, int R) {
  const int E = R % 8 == 0 ? R + (D + 7) / 8 * 8 : D + R;
  uint16_t* at = t.p + row * t.EP;
  for (int e = E + thread; e < t.EP; e += THREADS) {
    at[e] = 0;
    if constexpr (PL == 2) at[t.plane + e] = 0;
  }
}

// A thread's u-th chunk of eight columns of a tile of C rows: four side by side in a row, the next rows, then the next
// four: a wave's chunks are all rotated or mostly not.
template <int C, int THREADS>
struct LinItem {
  int row, d0;
  __device__ __forceinline__ explicit LinItem(int u, int tid = threadIdx.x) {
    const int t = tid + THREADS * u;
    row = (t >> 2) % C;
    d0 = ((t & 3) + 4 * (t / (4 * C))) * 8;
  }
};

// Operand of 16 rows x 32 columns, read across: lane l gets column n0 + l % 16 of rows r0 + 4 q + i, then r0 + 16 + 4 q + i
// (q = l / 16).  Row strides are an odd multiple of two 16-byte units, so that the eight rows of half a wave fall on different banks.
__device__ __forceinline__ u32x4 lin_across(const uint16_t* tile, int stride, int r0, int n0, int lane) {
  const int q = lane >> 4, j = lane & 15;
  const uint16_t* p = tile + (r0 + 4 * q + (j >> 2)) * stride + n0 + 4 * (j & 3);
  const u32x2 lo = lds_read_tr16(p), hi = lds_read_tr16(p + 16 * stride);
  return u32x4{lo[0], lo[1], hi[0], hi[1]};
}
// The same operand read along rows that keep their columns (two pieces), and that were permuted (one).
__device__ __forceinline__ u32x4 lin_along(const uint16_t* tile, int stride, int r0, int n0, int lane) {
  const uint16_t* p = tile + (r0 + (lane & 15)) * stride + n0 + 4 * (lane >> 4);
  const u32x2 lo = *reinterpret_cast<const u32x2*>(p), hi = *reinterpret_cast<const u32x2*>(p + 16);
  return u32x4{lo[0], lo[1], hi[0], hi[1]};
}
__device__ __forceinline__ u32x4 lin_along_placed(const uint16_t* tile, int stride, int r0, int n0, int lane) {
  return *reinterpret_cast<const u32x4*>(tile + (r0 + (lane & 15)) * stride + n0 + 8 * (lane >> 4));
}

// c + a b over operands of PA and PB bf16 parts; the product of two second parts is below what fp32 keeps of the others.
template <int PA, int PB>
__device__ __forceinline__ f32x4 lin_mfma(const u32x4* a, const u32x4* b, f32x4 c) {
#pragma unroll
  for (int i = PA - 1; i >= 0; --i)
#pragma unroll
    for (int j = PB - 1; j >= 0; --j)
      if (i + j < 2) c = BF16::mfma16(as_vec8<bf16x8>(a[i]), as_vec8<bf16x8>(b[j]), c);
  return c;
}

// Tile shapes: P columns of the contraction, NT columns of the result per workgroup, NW waves of SL columns each.
template <int PL_, int P_, int NT_, int NW_>
struct LinCfg {
  static constexpr int P = P_, NT = NT_, NW = NW_, SL = NT / NW, CT = SL / 16;
  static constexpr int kThreads = 64 * NW;
  static constexpr int PL = PL_;
  static constexpr int C = PL == 1 ? 64 : 32, KS = C / 32, IT = C / 16;
  static constexpr int XS = P + 8, YS = P + 16, ZS = NT + 16, AS = C + 8;
  static constexpr int TP = (C * (P / 8) + kThreads - 1) / kThreads, TZ = (C * (NT / 8) + kThreads - 1) / kThreads;
};

// Rows of P / NT that a call takes: dispatch over (P, NT), P for the contraction's columns, NT for the result's.
// Wide results go in tiles of 256 columns over eight waves; states of more than 256 rows leave room for 16 columns a wave.
// 65 to 96 columns run as 128 over four waves: six waves of 16 columns have nothing to skip, but a CU takes one such workgroup, not
// two (two waves on two of the SIMDs each time), and dq and dk of 2 x 8 heads x 4,096 rows of 64 + 32 columns took 70 us against 61.
template <int PL, template <typename> class Launch, typename... A>
hipError_t lin_dispatch(int pcols, int ncols, A&&... args) {
  const int p = pcols <= 64 ? 64 : pcols <= 96 ? 96 : pcols <= 128 ? 128 : pcols <= 256 ? 256 : 512;
  const int n = ncols <= 64 ? 64 : ncols <= 128 ? 128 : 256;
#define POPE_LIN_CASE(PP, NN, WW) return Launch<LinCfg<PL, PP, NN, WW>>::go(args...)
  if (p == 64) {
    if (n == 64) POPE_LIN_CASE(64, 64, 4);
    if (n == 128) POPE_LIN_CASE(64, 128, 4);
    POPE_LIN_CASE(64, 256, 8);
  }
  if (p == 96) {
    if (n == 64) POPE_LIN_CASE(96, 64, 4);
    if (n == 128) POPE_LIN_CASE(96, 128, 4);
    POPE_LIN_CASE(96, 256, 8);
  }
  if (p == 128) {
    if (n == 64) POPE_LIN_CASE(128, 64, 4);
    if (n == 128) POPE_LIN_CASE(128, 128, 4);
    POPE_LIN_CASE(128, 256, 8);
  }
  if (p == 256) {
    if (n == 64) POPE_LIN_CASE(256, 64, 4);
    if (n == 128) POPE_LIN_CASE(256, 128, 4);
    POPE_LIN_CASE(256, 256, 8);
  }
  POPE_LIN_CASE(512, 128, 8);
#undef POPE_LIN_CASE
}

}  // namespace pope
