// Expanded rows, states of the linear attention between segments, and the phases' gradients (gfx950).
//
//   states   the expanded rows (q_hat times the scale, k_hat, as bf16 parts: everything after reads them, forward and backward), and
//            what the rows of a segment add to the state behind it, sum_j g^(len-1-j) k_hat_j v_j^T; or, in reverse, to the gradient of
//            the state before it, sum_i g^(i+1) scale q_hat_i dO_i^T.  k_hat is weighted in fp32 and goes into the products as two
//            bf16 parts: 2^-16 of each, so that states can be handed on from call to call.
//   sums     the same sums from the expanded rows in memory, for the backward: states that only bf16 gradients read take one part
//   scan     S <- g^len S + sum, segment by segment; what a segment starts from goes where its sum was
//   phase    sums of the phases' gradients over segments (bias) and heads (freqs), in a fixed order
//
// Bound by memory, and by the sines and exponentials of the expansion: 32,768 rows of 8 heads, D 64, R 32, bf16, take 54-64 us (189 MB to and
// from HBM, 3 TB/s), the sums from expanded rows (2 x 4,096 of them) 11, a scan of 134 MB of states 28 (4.8 TB/s).
// Expanding rows where they are used instead cost more: the forward over those 32,768 rows took 86 us and its states 46, against 45 and
// 64 with the rows expanded here.  So did a launch of its own for the expansion: 20 us and 10 for the sums against 19 (2 x 4,096 rows).
#include <algorithm>
#include <type_traits>

#include "linear_dev.hpp"

namespace pope {

namespace {

// ---------------------------------------------------------------- states

// A workgroup's accumulators to its segment's place.
template <typename K>
__device__ __forceinline__ void lin_state_out(const LinStateParams& p, int at, int hk, int col0, const f32x4 (&W)[K::CT][K::P / 16]) {
  const LinCall& c = p.c;
  const int lane = threadIdx.x & 63, q4 = lane >> 4, l16 = lane & 15;
  float* to = p.states + ((int64_t)at * c.Hk + hk) * c.E * c.Dv;
#pragma unroll
  for (int ct = 0; ct < K::CT; ++ct) {
    const int col = col0 + 16 * ct + l16;
#pragma unroll
    for (int s = 0; s < K::P / 16; ++s)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * s + 4 * q4 + r;
        if (row < c.E && col < c.Dv) to[(int64_t)row * c.Dv + col] = W[ct][s][r];
      }
  }
}

// A chunk of a row and its angles, as they are in memory.  FAST: whole units; then nothing decides whether the loads happen (a
// branch around a load waits for it), and places past the end are moved to the last ones.
template <int PL>
struct LinIn {
  LinRaw<PL> x;
  f32x4 f[2];
};
template <int PL, bool FAST>
__device__ __forceinline__ LinIn<PL> lin_in(const LinCall& c, const LinRows& r, const char* base, const char* f_base, uint32_t at, int d0) {
  LinIn<PL> o;
  o.f[0] = o.f[1] = f32x4{0.f, 0.f, 0.f, 0.f};
  o.x = lin_load8<PL>(r, base, at * lin_step(r), FAST ? min(d0, c.D - 8) : d0, FAST);
  if (!c.R) return o;
  const float* fr = reinterpret_cast<const float*>(f_base + (uint32_t)(at * (uint32_t)c.f_s[1] * 4));
  if constexpr (FAST) {
    const int d = min(d0, c.R - 8);
    o.f[0] = *reinterpret_cast<const f32x4*>(fr + d);
    o.f[1] = *reinterpret_cast<const f32x4*>(fr + d + 4);
  } else {
    lin_angles8(fr, d0, c.R, false, o.f);
  }
  return o;
}
__device__ __forceinline__ bool lin_fast(const LinCall& c, const LinRows& r) { return r.vec && (c.f_vec || !c.R); }
__device__ __forceinline__ char* lin_angle_base(const LinCall& c, int batch, int64_t row) {
  return c.R ? lin_uniform(c.freqs + (int64_t)batch * c.f_s[0] + row * c.f_s[1]) : nullptr;
}

// The queries of a segment and head, expanded: four threads a row, two rows and two chunks of each at once.  A workgroup has every
// parts-th 64 columns: where one workgroup fills a CU, queries are small pieces behind the keys' long ones (D 256, R 256, 2 x 2,048 rows:
// 94 us whole, 86 so; with four waves, 16 heads on 4 of D 128, R 64, 27.5 whole, 30 so).
template <int PL, int THREADS, bool FAST>
__device__ __forceinline__ void lin_expand_queries(const LinCall& c, const LinSeg& seg, int hq, int part, int parts) {
  const int tid = threadIdx.x, per = (c.D + 7) / 8;
  constexpr int kRows = THREADS / 4;
  for (int r0 = 0; r0 < seg.len; r0 += 2 * kRows) {
    const char* base = lin_base(c.q, seg.batch, hq, seg.row0 + r0);
    const char* f_base = lin_angle_base(c, seg.batch, seg.row0 + r0);
    const int64_t to = ((int64_t)seg.batch * c.Hq + hq) * c.seqs.N + seg.row0 + r0;
    const int left = seg.len - r0;
    for (int u0 = 8 * part + (tid & 3); u0 - (tid & 3) < per; u0 += 8 * parts) {
      LinIn<PL> in[2][2];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int r = (tid >> 2) + j * kRows, u = u0 + 4 * k;
          if (FAST || (r < left && u < per)) in[j][k] = lin_in<PL, FAST>(c, c.q, base, f_base, min(r, left - 1), 8 * u);
        }
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int r = (tid >> 2) + j * kRows, u = u0 + 4 * k;
          if (r < left && u < per) {
            float a[8], b[8];
            lin_polar8<PL>(in[j][k].x, c.q.type, in[j][k].f, 8 * u, c.R, c.scale, nullptr, a, b);
            lin_hat_put<PL>(c.qh, to + r, 8 * u, c.D, c.R, a, b);
          }
          __builtin_amdgcn_sched_barrier(0);   // one expansion at a time: side by side they take all registers
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = (tid >> 2) + j * kRows;
      if (r < left && part == 0) lin_hat_tail<PL, 4>(c.qh, to + r, tid & 3, c.D, c.R);
    }
  }
}

// p.states may be null: the expanded rows only.
template <typename K>
__global__ __launch_bounds__(K::kThreads, 1) void linear_state_kernel(LinStateParams p) {
  constexpr int NT = K::NT, CT = K::CT, PL = K::PL, C = K::C, KS = K::KS, ST = K::P / 32;
  __shared__ __attribute__((aligned(16))) uint16_t lds[2 * C * K::YS + PL * C * K::ZS];
  __shared__ float turns[256];
  const LinCall& c = p.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), q4 = lane >> 4, l16 = lane & 15;
  if ((int)blockIdx.x >= p.key_wgs) {
    const int part = (blockIdx.x - p.key_wgs) % p.q_parts, wg = (blockIdx.x - p.key_wgs) / p.q_parts, at = wg / c.Hq;
    const LinSeg seg = lin_segment(c.seqs, at);
    if (seg.seq < 0) return;
    if (lin_fast(c, c.q)) lin_expand_queries<PL, K::kThreads, true>(c, seg, wg - at * c.Hq, part, p.q_parts);
    else lin_expand_queries<PL, K::kThreads, false>(c, seg, wg - at * c.Hq, part, p.q_parts);
    return;
  }
  const int wg = blockIdx.x, tile = wg % p.tiles, rest = wg / p.tiles, hk = rest % c.Hk, at = rest / c.Hk;
  const LinSeg seg = lin_segment(c.seqs, at);
  if (seg.seq < 0) return;
  const LinTile Y{lds, K::YS, C * K::YS}, Z{lds + 2 * C * K::YS, K::ZS, C * K::ZS};
  for (int i = tid; i < (int)sizeof(lds) / 16; i += K::kThreads) reinterpret_cast<u32x4*>(lds)[i] = u32x4{0, 0, 0, 0};
  const bool rev = p.reverse != 0;
  if (!rev)
    for (int d = tid; d < c.R; d += K::kThreads) turns[d] = lin_turns(lin_bias(c, hk, d));
  const float lg = lin_log2(c, hk);
  const int n0 = tile * NT, col0 = wave * K::SL, steps = (c.E + 31) / 32, G = rev ? c.G : 1;
  const bool busy = n0 + col0 < c.Dv;
  f32x4 W[CT][2 * ST];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
#pragma unroll
    for (int s = 0; s < 2 * ST; ++s) W[ct][s] = f32x4{0.f, 0.f, 0.f, 0.f};
  const LinRows yr = rev ? c.q : c.k, zr = rev ? c.g : c.v;
  const float* bias = rev ? nullptr : turns;
  const int ty = (C * ((c.D + 31) / 32 * 4) + K::kThreads - 1) / K::kThreads;
  const int tz = (C * ((min(NT, c.Dv - n0) + 31) / 32 * 4) + K::kThreads - 1) / K::kThreads;
  typedef LinItem<C, K::kThreads> Item;
  const uint8_t* mask = rev || !c.mask ? nullptr : c.mask + (int64_t)seg.batch * c.mask_sb + seg.row0;
  // a turn's chunks of a tile, two at once
  const auto turn_y = [&](auto fast, int t0, int h, int u0) {
    constexpr bool kFast = decltype(fast)::value;
    const char* base = lin_base(yr, seg.batch, h, seg.row0 + t0);
    const char* f_base = lin_angle_base(c, seg.batch, seg.row0 + t0);
    const int left = seg.len - t0;
    LinIn<PL> in[2];
    uint32_t live[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const Item i(u0 + k);
      const int at = min(i.row, left - 1);
      if (kFast || i.d0 < c.D) in[k] = lin_in<PL, kFast>(c, yr, base, f_base, at, i.d0);
      live[k] = mask ? (uint32_t)mask[t0 + at] : 1u;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const Item i(u0 + k);
      const bool there = i.row < left, keep = !rev && tile == 0 && there;
      const int64_t to = ((int64_t)seg.batch * c.Hk + hk) * c.seqs.N + seg.row0 + t0 + i.row;
      if (keep && i.d0 < 32) lin_hat_tail<PL, 4>(c.kh, to, i.d0 / 8, c.D, c.R);
      if (i.d0 < c.D) {
        float a[8], b[8];
        lin_polar8<PL>(in[k].x, yr.type, in[k].f, i.d0, c.R, rev ? c.scale : 1.f, bias, a, b);
        if (!there || !live[k])
#pragma unroll
          for (int j = 0; j < 8; ++j) a[j] = b[j] = 0.f;
        if (keep) lin_hat_put<PL>(c.kh, to, i.d0, c.D, c.R, a, b);
        if (p.states) {
          const float w = there ? lin_power(lg, rev ? t0 + i.row + 1 : left - 1 - i.row) : 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) a[j] *= w, b[j] *= w;
          lin_place8(i.d0, c.D, c.R, a, b, [&](int e, const float* v) { lin_put8<2, false>(Y, i.row, e, v); },
                     [&](int e, float v) { lin_put1<2, false>(Y, i.row, e, v); });
        }
      }
      __builtin_amdgcn_sched_barrier(0);   // one expansion at a time: side by side they take all registers
    }
  };
  constexpr int kZ = 2;   // chunks of values that are loaded in front of the keys'
  LinRaw<PL> zin[kZ];
  uint32_t zlive[kZ];
  const auto get_z = [&](auto fast, int t0, int h, int u, LinRaw<PL>& x, uint32_t& live) {
    constexpr bool kFast = decltype(fast)::value;
    const char* base = lin_base(zr, seg.batch, h, seg.row0 + t0);
    const Item i(u);
    const int at = min(i.row, seg.len - t0 - 1), d0 = n0 + i.d0;
    x = LinRaw<PL>{};
    if (kFast || (i.d0 < NT && d0 < c.Dv)) x = lin_load8<PL>(zr, base, at * lin_step(zr), kFast ? min(d0, c.Dv - 8) : d0, kFast);
    live = mask ? (uint32_t)mask[t0 + at] : 1u;
  };
  const auto put_z = [&](int t0, int u, LinRaw<PL> x, uint32_t live) {
    const Item i(u);
    if (i.d0 >= NT || n0 + i.d0 >= c.Dv) return;
    if (i.row >= seg.len - t0 || !live) x = LinRaw<PL>{};
    lin_put_plain<PL, false>(Z, i.row, i.d0, x, zr.type);
  };
  const bool fast_y = lin_fast(c, yr), fast_z = zr.vec;
  for (int t0 = 0; t0 < seg.len; t0 += C)
    for (int g = 0; g < G; ++g) {
      const int h = rev ? g * c.Hk + hk : hk;
      if (p.states) {
#pragma unroll
        for (int u = 0; u < kZ; ++u) {
          if (fast_z) get_z(std::true_type{}, t0, h, u, zin[u], zlive[u]);
          else get_z(std::false_type{}, t0, h, u, zin[u], zlive[u]);
        }
      }
      __syncthreads();   // nothing reads the tiles any more
#pragma unroll 1
      for (int u = 0; u < ty; u += 2) {
        if (fast_y) turn_y(std::true_type{}, t0, h, u);
        else turn_y(std::false_type{}, t0, h, u);
      }
      if (!p.states) continue;
#pragma unroll
      for (int u = 0; u < kZ; ++u) put_z(t0, u, zin[u], zlive[u]);
#pragma unroll 2
      for (int u = kZ; u < tz; ++u) {
        LinRaw<PL> x;
        uint32_t live;
        if (fast_z) get_z(std::true_type{}, t0, h, u, x, live);
        else get_z(std::false_type{}, t0, h, u, x, live);
        put_z(t0, u, x, live);
      }
      __syncthreads();
      if (busy) {
        u32x4 za[CT][KS][PL];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
          for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int l = 0; l < PL; ++l) za[ct][s][l] = lin_across(Z.p + l * Z.plane, K::ZS, 32 * s, col0 + 16 * ct, lane);
#pragma unroll
        for (int e = 0; e < 2 * ST; ++e)
          if (e < 2 * steps) {
#pragma unroll
            for (int s = 0; s < KS; ++s) {
              u32x4 ya[2];
#pragma unroll
              for (int l = 0; l < 2; ++l) ya[l] = lin_across(Y.p + l * Y.plane, K::YS, 32 * s, 16 * e, lane);
#pragma unroll
              for (int ct = 0; ct < CT; ++ct) W[ct][e] = lin_mfma<2, PL>(ya, za[ct][s], W[ct][e]);
            }
          }
      }
    }
  if (busy && p.states) lin_state_out<K>(p, at, hk, n0 + col0, W);
}

// From the expanded rows.  EXACT: both factors as two parts (rows that are held as two).
template <typename K, bool EXACT>
__global__ __launch_bounds__(K::kThreads, K::P <= 128 && K::NT <= 128 ? 2 : K::NW / 4) void linear_sum_kernel(LinStateParams p) {
  constexpr int NT = K::NT, CT = K::CT, PL = K::PL, PY = EXACT ? 2 : 1, C = K::C, KS = K::KS, ST = K::P / 32;
  __shared__ __attribute__((aligned(16))) uint16_t lds[PY * C * K::YS + PL * C * K::ZS];
  __shared__ __attribute__((aligned(16))) float weight[C];
  const LinCall& c = p.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), q4 = lane >> 4, l16 = lane & 15;
  const int wg = blockIdx.x, tile = wg % p.tiles, rest = wg / p.tiles, hk = rest % c.Hk, at = rest / c.Hk;
  const LinSeg seg = lin_segment(c.seqs, at);
  if (seg.seq < 0) return;
  const LinTile Y{lds, K::YS, C * K::YS}, Z{lds + PY * C * K::YS, K::ZS, C * K::ZS};
  for (int i = tid; i < (int)sizeof(lds) / 16; i += K::kThreads) reinterpret_cast<u32x4*>(lds)[i] = u32x4{0, 0, 0, 0};
  const bool rev = p.reverse != 0;
  const float lg = lin_log2(c, hk);
  const int n0 = tile * NT, col0 = wave * K::SL, steps = (c.E + 31) / 32, G = rev ? c.G : 1;
  const bool busy = n0 + col0 < c.Dv;
  f32x4 W[CT][2 * ST];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
#pragma unroll
    for (int s = 0; s < 2 * ST; ++s) W[ct][s] = f32x4{0.f, 0.f, 0.f, 0.f};
  const LinHat yh = rev ? c.qh : c.kh;
  const LinRows zr = rev ? c.g : c.v;
  typedef LinItem<C, K::kThreads> Item;
  const uint8_t* mask = rev || !c.mask ? nullptr : c.mask + (int64_t)seg.batch * c.mask_sb + seg.row0;
  struct InY { u32x4 w[PY]; };
  struct InZ { LinRaw<PL> x; uint32_t live; };
  // loads that nothing decides about (a branch around a load waits for it): rows behind the segment are the last one's again, what
  // the mask leaves out is read too, and becomes zeros on the way into LDS
  const auto get_y = [&](int it, int u) {
    const Item i(u);
    const int t0 = it / G * C, h = rev ? it % G * c.Hk + hk : hk, at = min(i.row, seg.len - 1 - t0);
    const char* base = lin_uniform(yh.p + (((int64_t)seg.batch * yh.H + h) * c.seqs.N + seg.row0 + t0) * yh.EP);
    InY r;
#pragma unroll
    for (int l = 0; l < PY; ++l) r.w[l] = *reinterpret_cast<const u32x4*>(base + l * 2 * yh.plane + (uint32_t)((at * yh.EP + min(i.d0, yh.EP - 8)) * 2));
    return r;
  };
  const auto get_z = [&](auto fast, int it, int u) {
    constexpr bool kFast = decltype(fast)::value;
    const Item i(u);
    const int t0 = it / G * C, h = rev ? it % G * c.Hk + hk : hk, at = min(i.row, seg.len - 1 - t0), d0 = n0 + i.d0;
    const char* base = lin_base(zr, seg.batch, h, seg.row0 + t0);
    InZ r;
    r.x = LinRaw<PL>{};
    if (kFast || d0 < c.Dv) r.x = lin_load8<PL>(zr, base, at * lin_step(zr), kFast ? min(d0, c.Dv - 8) : d0, kFast);
    r.live = mask ? (uint32_t)mask[t0 + at] : 1u;
    return r;
  };
  const auto put_y = [&](int it, int u, InY r) {
    const Item i(u);
    if (i.d0 >= yh.EP) return;
    if (it / G * C + i.row >= seg.len)
#pragma unroll
      for (int l = 0; l < PY; ++l) r.w[l] = u32x4{0, 0, 0, 0};
    lin_put_parts<PY, false>(Y, i.row, i.d0, r.w);
  };
  const auto put_z = [&](int it, int u, InZ r) {
    const Item i(u);
    if (i.d0 >= NT || n0 + i.d0 >= c.Dv) return;
    if (it / G * C + i.row >= seg.len || !r.live) r.x = LinRaw<PL>{};
    lin_put_plain<PL, false>(Z, i.row, i.d0, r.x, zr.type);
  };
  const bool fast = zr.vec;
  constexpr bool kAhead = K::P <= 128 && NT <= 128;
  constexpr int kTY = kAhead ? K::TP : 0, kTZ = kAhead ? K::TZ : 0;
  InY yin[kTY + 1];
  InZ zin[kTZ + 1];
  const auto load = [&](int it) {
#pragma unroll
    for (int u = 0; u < kTY; ++u) yin[u] = get_y(it, u);
#pragma unroll
    for (int u = 0; u < kTZ; ++u) {
      if (fast) zin[u] = get_z(std::true_type{}, it, u);
      else zin[u] = get_z(std::false_type{}, it, u);
    }
  };
  const int all = (seg.len + C - 1) / C * G;
  load(0);
  for (int it = 0; it < all; ++it) {
    __syncthreads();   // nothing reads the tiles any more
    for (int t = tid; t < C; t += K::kThreads) {
      const int at_t = it / G * C + t;
      weight[t] = at_t < seg.len ? lin_power(lg, rev ? at_t + 1 : seg.len - 1 - at_t) : 0.f;
    }
    if constexpr (kAhead) {
#pragma unroll
      for (int u = 0; u < kTY; ++u) put_y(it, u, yin[u]);
#pragma unroll
      for (int u = 0; u < kTZ; ++u) put_z(it, u, zin[u]);
      if (it + 1 < all) load(it + 1);
    } else {
      const int ty = (C * (yh.EP / 8) + K::kThreads - 1) / K::kThreads;
      const int tz = (C * ((min(NT, c.Dv - n0) + 31) / 32 * 4) + K::kThreads - 1) / K::kThreads;
#pragma unroll 4
      for (int u = 0; u < ty; ++u) put_y(it, u, get_y(it, u));
#pragma unroll 4
      for (int u = 0; u < tz; ++u) put_z(it, u, fast ? get_z(std::true_type{}, it, u) : get_z(std::false_type{}, it, u));
    }
    __syncthreads();
    if (busy) {
      u32x4 za[CT][KS][PY];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const f32x4 w0 = *reinterpret_cast<const f32x4*>(weight + 32 * s + 4 * q4), w1 = *reinterpret_cast<const f32x4*>(weight + 32 * s + 16 + 4 * q4);
          float v[8];
          unpack8<BF16>(lin_across(Z.p, K::ZS, 32 * s, col0 + 16 * ct, lane), v);
          if constexpr (PL == 2) {
            float v2[8];
            unpack8<BF16>(lin_across(Z.p + Z.plane, K::ZS, 32 * s, col0 + 16 * ct, lane), v2);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += v2[j];
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] *= w0[j], v[4 + j] *= w1[j];
          u32x2 lo[PY], hi[PY];
          lin_pack4<PY>(f32x4{v[0], v[1], v[2], v[3]}, lo);
          lin_pack4<PY>(f32x4{v[4], v[5], v[6], v[7]}, hi);
#pragma unroll
          for (int l = 0; l < PY; ++l) za[ct][s][l] = u32x4{lo[l][0], lo[l][1], hi[l][0], hi[l][1]};
        }
#pragma unroll
      for (int e = 0; e < 2 * ST; ++e)
        if (e < 2 * steps) {
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            u32x4 ya[PY];
#pragma unroll
            for (int l = 0; l < PY; ++l) ya[l] = lin_across(Y.p + l * Y.plane, K::YS, 32 * s, 16 * e, lane);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) W[ct][e] = lin_mfma<PY, PY>(ya, za[ct][s], W[ct][e]);
          }
        }
    }
  }
  if (busy) lin_state_out<K>(p, at, hk, n0 + col0, W);
}

template <typename K>
struct StateLaunch {
  static hipError_t go(LinStateParams p, hipStream_t s) {
    p.tiles = p.states ? (p.c.Dv + K::NT - 1) / K::NT : 1;
    const int64_t keys = (int64_t)p.c.seqs.T * p.c.Hk * p.tiles, heads = p.reverse ? 0 : (int64_t)p.c.seqs.T * p.c.Hq;
    p.q_parts = K::NW == 8 ? (p.c.D + 63) / 64 : 1;
    const int64_t n = keys + heads * p.q_parts;
    if (n >= ((int64_t)1 << 22)) return hipErrorInvalidValue;
    p.key_wgs = (int)keys;
    return launch_named("linear_states", linear_state_kernel<K>, dim3((unsigned)n), dim3(K::kThreads), s, p);
  }
};

template <bool EXACT>
struct SumLaunch {
  template <typename K>
  struct Of {
    static hipError_t go(LinStateParams p, hipStream_t s) {
      p.tiles = (p.c.Dv + K::NT - 1) / K::NT;
      const int64_t n = (int64_t)p.c.seqs.T * p.c.Hk * p.tiles;
      if (n >= ((int64_t)1 << 22)) return hipErrorInvalidValue;
      return launch_named("linear_sums", linear_sum_kernel<K, EXACT>, dim3((unsigned)n), dim3(K::kThreads), s, p);
    }
  };
};

// ---------------------------------------------------------------- scan and phase

constexpr int kScanAhead = 8;   // segments whose sums are loaded ahead of the sum over them

__global__ __launch_bounds__(256) void linear_scan_kernel(LinScanParams p) {
  const LinCall& c = p.c;
  const int per = c.E * c.Dv, blocks = (per + 255) / 256, hk = blockIdx.y, seq = blockIdx.x / blocks;
  const int i = (blockIdx.x - seq * blocks) * 256 + threadIdx.x;
  int first, row0 = 0, rows = c.seqs.N;
  if (c.seqs.cu) first = lin_first(c.seqs, seq, &row0, &rows);
  else first = seq * c.seqs.M;
  if (i >= per) return;
  const int L = c.seqs.L, count = min((rows + L - 1) / L, c.seqs.T - first);
  const float lg = lin_log2(c, hk);
  const int64_t own = ((int64_t)seq * c.Hk + hk) * per + i, step = (int64_t)c.Hk * per;
  float* at = p.states + ((int64_t)first * c.Hk + hk) * per + i;
  float S = p.first ? p.first[own] : 0.f;
  const float whole = lin_power(lg, L), part = lin_power(lg, rows - (count - 1) * L);   // of a segment's rows, of the last one's
  for (int m0 = 0; m0 < count; m0 += kScanAhead) {
    float u[kScanAhead];
#pragma unroll
    for (int k = 0; k < kScanAhead; ++k)
      if (m0 + k < count) u[k] = at[(p.reverse ? count - 1 - m0 - k : m0 + k) * step];
#pragma unroll
    for (int k = 0; k < kScanAhead; ++k)
      if (m0 + k < count) {
        const int m = p.reverse ? count - 1 - m0 - k : m0 + k;
        at[m * step] = S;
        S = fmaf(m == count - 1 ? part : whole, S, u[k]);
      }
  }
  if (p.last) p.last[own] = S;
}

// A thread per (bias row, dim) and quarter of the segments.
__global__ __launch_bounds__(256) void linear_dbias_kernel(LinPhaseParams p) {
  __shared__ float red[4][64];
  const LinCall& c = p.c;
  const int d = blockIdx.x * 64 + (threadIdx.x & 63), q = threadIdx.x >> 6, h0 = blockIdx.y;
  float sum = 0.f;
  if (d < c.R)
    for (int h = h0; h < c.Hk; h += p.Hb)
#pragma unroll 4
      for (int s = q; s < c.seqs.T; s += 4) sum += p.part[((int64_t)s * c.Hk + h) * c.R + d];
  red[q][threadIdx.x & 63] = sum;
  __syncthreads();
  if (q == 0 && d < c.R) {
    const float v = (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
    const int64_t at = (int64_t)h0 * c.R + d;
    if (c.bias_type == 0) static_cast<float*>(p.dbias)[at] = v;
    else static_cast<uint16_t*>(p.dbias)[at] = c.bias_type == 1 ? F16::bits(v) : BF16::bits(v);
  }
}

// A thread per (table batch, row, dim).
__global__ __launch_bounds__(256) void linear_dfreqs_kernel(LinPhaseParams p) {
  const LinCall& c = p.c;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, per = (int64_t)c.seqs.N * c.R;
  if (i >= per) return;
  const int fb = blockIdx.y, batches = c.seqs.cu ? 1 : c.seqs.B;
  float sum = 0.f;
  for (int b = fb; b < batches; b += p.Fb) {
    for (int h = 0; h < c.Hq; ++h) sum += p.dphase_q[((int64_t)b * c.Hq + h) * per + i];
    for (int h = 0; h < c.Hk; ++h) sum += p.dphase_k[((int64_t)b * c.Hk + h) * per + i];
  }
  const int64_t n = i / c.R, d = i - n * c.R;
  p.dfreqs[(int64_t)fb * p.df_s[0] + n * p.df_s[1] + d] = sum;
}

}  // namespace

// Columns of values for a workgroup: narrower tiles, whose expanded rows are read or made again, where wide ones leave CUs without work.
int sum_cols(const LinCall& c) {
  int n = c.Dv <= 64 ? 64 : c.Dv <= 128 ? 128 : 256;
  while (n > 64 && (int64_t)c.seqs.T * c.Hk * ((c.Dv + n - 1) / n) < 256) n /= 2;
  return std::min(n, c.Dv);
}

hipError_t launch_linear_states(const LinStateParams& p, hipStream_t s) {
  const int n = sum_cols(p.c);
  return p.c.split ? lin_dispatch<kTwo, StateLaunch>(p.c.E, n, p, s) : lin_dispatch<kOne, StateLaunch>(p.c.E, n, p, s);
}

hipError_t launch_linear_sums(const LinStateParams& p, hipStream_t s) {
  const int n = sum_cols(p.c);
  return p.c.split ? lin_dispatch<kTwo, SumLaunch<true>::template Of>(p.c.E, n, p, s) : lin_dispatch<kOne, SumLaunch<false>::template Of>(p.c.E, n, p, s);
}

hipError_t launch_linear_scan(const LinScanParams& p, hipStream_t s) {
  const int64_t n = (int64_t)((p.c.E * p.c.Dv + 255) / 256) * p.c.seqs.B;
  if (n >= ((int64_t)1 << 22)) return hipErrorInvalidValue;
  return launch_named("linear_scan", linear_scan_kernel, dim3((unsigned)n, p.c.Hk), dim3(256), s, p);
}

hipError_t launch_linear_phase(const LinPhaseParams& p, hipStream_t s) {
  if (p.dbias) {
    const hipError_t e = launch_named("linear_dbias", linear_dbias_kernel, dim3((p.c.R + 63) / 64, p.Hb), dim3(256), s, p);
    if (e != hipSuccess) return e;
  }
  if (!p.dfreqs) return hipSuccess;
  const int64_t n = ((int64_t)p.c.seqs.N * p.c.R + 255) / 256;
  if (n >= ((int64_t)1 << 23)) return hipErrorInvalidValue;
  return launch_named("linear_dfreqs", linear_dfreqs_kernel, dim3((unsigned)n, p.Fb), dim3(256), s, p);
}

}  // namespace pope
