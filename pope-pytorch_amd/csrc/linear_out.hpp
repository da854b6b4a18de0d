// Outputs and gradients of the linear attention with head decays (gfx950).
//
// With expanded rows q_hat, k_hat and g = exp(log_decay), rows i of a sequence:
//   S_i = g S_(i-1) + k_hat_i v_i^T,  o_i = scale S_i^T q_hat_i
// and with G_i the gradient of S_i, G_i = g G_(i+1) + scale q_hat_i dO_i^T (behind the last row: the final state's gradient):
//   dq_hat_i = scale S_i dO_i,  dk_hat_i = G_i v_i,  dv_i = G_i^T k_hat_i
// All four are one computation on rows x, y, z, in the rows' order or, for the last two, the reverse:
//   out_i = sum_{j <= i} g^(i-j) (x_i . y_j) z_j + g^(i+a) W^T x_i
//   kind    x        y        z        W (P x columns)        a
//   out     q_hat    k_hat    v        S behind the segment before          1
//   dq      dO       v        k_hat    its transpose                        1
//   dk      v        dO       q_hat    the transpose of g G                 0
//   dv      k_hat    q_hat    dO       g G of the segment behind            0
// A workgroup takes a segment of rows of one head in chunks of C, with W in registers as fp32 accumulators: the products of
// a chunk's rows with each other (C x C, weighted by powers of g, through LDS), with W, and the chunk's own part of W for the next
// chunk.  W's accumulators are in the order in which a product reads an operand, so W goes from one to the next without
// leaving its registers.
//
// Rounding: x, y, z, the weighted C x C products and W as an operand are bf16: one part for bf16 rows (each is off by at most 2^-9,
// as the output is by its own rounding), the sum of two for fp16 rows (2^-17).  W itself, all sums and the powers of g are
// fp32.
#pragma once
#include "linear_dev.hpp"

namespace pope {

template <typename T, typename K, int KIND>
__device__ __forceinline__ void lin_out_job(const LinOutParams& p, int wg, char* smem) {
  constexpr int kind = KIND, which = KIND == kLinDk ? 1 : 0;
  constexpr int P = K::P, NT = K::NT, CT = K::CT, PL = K::PL, C = K::C, KS = K::KS, IT = K::IT, ST = P / 32;
  constexpr int kThreads = K::kThreads;
  const LinCall& c = p.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), q4 = lane >> 4, l16 = lane & 15;
  constexpr bool by_query = kind == kLinOut || kind == kLinDq;   // x changes with the query heads of the key head; else y and z do
  constexpr bool rev = !by_query;

  // tile of columns fastest, then head, then segment: neighbours share their rows
  const int groups = by_query ? c.G / p.heads_per : 1, heads = c.Hk * groups;
  const int tiles = p.tiles;
  const int tile = wg % tiles, rest = wg / tiles, head = rest % heads, at = rest / heads;
  const int hk = head % c.Hk, g0 = head / c.Hk * p.heads_per, ng = by_query ? p.heads_per : c.G;
  const LinRows out = p.out[which];
  const int ncols = kind == kLinOut || kind == kLinDv ? c.Dv : c.E;          // columns of the result, as computed
  const int pcols = kind == kLinOut || kind == kLinDv ? c.E : c.Dv;          // of the contraction
  const int n0 = tile * NT;
  constexpr bool chain = kind == kLinDq || kind == kLinDk;
  const int out_cols = out.cols;

  if (c.seqs.cu && at == c.seqs.T) {   // rows outside every sequence: zeros
    if (tile) return;
    const int lo = lin_bound(c.seqs, 0), hi = lin_bound(c.seqs, c.seqs.B);
    for (int64_t it = tid; it < (int64_t)(lo + c.seqs.N - hi) * out_cols; it += kThreads) {
      const int r = (int)(it / out_cols), d = (int)(it - (int64_t)r * out_cols), row = r < lo ? r : hi + r - lo;
      for (int g = 0; g < (by_query ? ng : 1); ++g) {
        const int h = by_query ? (g0 + g) * c.Hk + hk : hk;
        out.p[(int64_t)h * out.s[1] + (int64_t)row * out.s[2] + d] = 0;
        if (chain && p.dphase[which] && d < c.R) p.dphase[which][((int64_t)h * c.seqs.N + row) * c.R + d] = 0.f;
      }
    }
    return;
  }
  const LinSeg seg = lin_segment(c.seqs, at);
  if (kind == kLinDk && p.dbias && seg.seq < 0) {
    for (int d = tid; d < c.R; d += kThreads) p.dbias[((int64_t)at * c.Hk + hk) * c.R + d] = 0.f;
  }
  if (seg.seq < 0) return;

  uint16_t* lds = reinterpret_cast<uint16_t*>(smem);
  const LinTile X{lds, K::XS, C * K::XS};
  const LinTile Y{X.p + PL * X.plane, K::YS, C * K::YS};
  const LinTile Z{Y.p + PL * Y.plane, K::ZS, C * K::ZS};
  const LinTile A{Z.p + PL * Z.plane, K::AS, C * K::AS};
  float* turns = reinterpret_cast<float*>(A.p + PL * A.plane);   // 256
  int* odd = reinterpret_cast<int*>(turns + 256);                // z of this chunk that are not finite; two, by turns
  constexpr int kTileBytes = PL * (C * (K::XS + K::YS + K::ZS + K::AS)) * 2;
  for (int i = tid; i < kTileBytes / 16; i += kThreads) reinterpret_cast<u32x4*>(smem)[i] = u32x4{0, 0, 0, 0};
  if (tid < 2) odd[tid] = 0;
  for (int d = tid; d < c.R; d += kThreads) turns[d] = lin_turns(c.bias[hk * c.bias_sh + d]);

  const float lg = lin_log2(c, hk);
  const int a = rev ? 0 : 1;
  const int chunks = (seg.len + C - 1) / C;
  const int col0 = wave * K::SL;                    // the wave's columns in the tile
  const bool busy = n0 + col0 < ncols;
  const int steps = (pcols + 31) / 32;

  // W: accumulators of 16-row tiles 4 q4 + i x columns l16
  f32x4 W[CT][2 * ST];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
#pragma unroll
    for (int s = 0; s < 2 * ST; ++s) W[ct][s] = f32x4{0.f, 0.f, 0.f, 0.f};
  {
    const float* from = p.states[rev] ? p.states[rev] + ((int64_t)at * c.Hk + hk) * c.E * c.Dv
                        : p.first[rev] ? p.first[rev] + ((int64_t)seg.seq * c.Hk + hk) * c.E * c.Dv : nullptr;
    if (from && busy) {
      const int64_t rs = chain ? 1 : c.Dv, cs = chain ? c.Dv : 1;   // transposed where the result has expanded columns
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        const int col = n0 + col0 + 16 * ct + l16;
#pragma unroll
        for (int s = 0; s < 2 * ST; ++s)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int row = 16 * s + 4 * q4 + r;
            if (row < pcols && col < ncols) W[ct][s][r] = from[row * rs + col * cs];
          }
      }
    }
  }
  const float keep = lin_power(lg, C);
  // weights of a chunk's rows in the next state, in the order of operands
  float wz[KS][8];
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int j = 0; j < 8; ++j) wz[s][j] = lin_power(lg, C - a - (32 * s + 16 * (j >> 2) + 4 * q4 + (j & 3)));
  float dbsum[CT][2];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) dbsum[ct][0] = dbsum[ct][1] = 0.f;

  const auto row_of = [&](int t) { return seg.row0 + (rev ? seg.len - 1 - t : t); };   // t: of the segment, in the job's order
  typedef LinItem<C, kThreads> Item;
  const LinRows xr = kind == kLinOut ? c.q : kind == kLinDq ? c.g : kind == kLinDk ? c.v : c.k;
  const LinRows yr = kind == kLinOut ? c.k : kind == kLinDq ? c.v : kind == kLinDk ? c.g : c.q;
  const LinRows zr = kind == kLinOut ? c.v : kind == kLinDq ? c.k : kind == kLinDk ? c.q : c.g;
  constexpr bool xy_polar = !chain, z_polar = chain;
  constexpr bool x_key = kind == kLinDk || kind == kLinDv, yz_key = !x_key;   // rows that the mask may leave out
  const auto kept = [&](int row) { return !c.mask || c.mask[(int64_t)seg.batch * c.mask_sb + row] != 0; };
  // A thread's chunks of the tiles: read from memory ...
  struct In { u32x4 x, y; f32x4 f[2]; bool lx, ly; };
  struct InZ { u32x4 z; f32x4 f[2]; bool live; };
  struct Turn { int t0, hq; bool lx, lyz; };
  const auto turn_of = [&](int it) {
    const int ch = it / ng, g = it - ch * ng;
    return Turn{ch * C, (g0 + g) * c.Hk + hk, by_query || g == 0, !by_query || g == 0};
  };
  const auto load_xy = [&](const Turn& n, int u) {
    const Item i(u);
    In r;
    r.x = r.y = u32x4{0, 0, 0, 0};
    r.f[0] = r.f[1] = f32x4{0.f, 0.f, 0.f, 0.f};
    r.lx = r.ly = false;
    if (n.t0 + i.row < seg.len && i.d0 < xr.cols) {   // x and y have as many columns
      const int row = row_of(n.t0 + i.row);
      const bool k = kept(row);
      r.lx = !x_key || k;
      r.ly = !yz_key || k;
      if (n.lx && r.lx) r.x = lin_load8(xr.p + (int64_t)seg.batch * xr.s[0] + (int64_t)(by_query ? n.hq : hk) * xr.s[1] + (int64_t)row * xr.s[2], i.d0, xr.cols, xr.vec);
      if (n.lyz && r.ly) r.y = lin_load8(yr.p + (int64_t)seg.batch * yr.s[0] + (int64_t)(by_query ? hk : n.hq) * yr.s[1] + (int64_t)row * yr.s[2], i.d0, yr.cols, yr.vec);
      if (xy_polar && c.R) lin_angles8(lin_angle_row(c, seg.batch, row), i.d0, c.R, c.f_vec, r.f);
    }
    return r;
  };
  const auto load_z = [&](const Turn& n, int u) {
    const Item i(u);
    InZ r;
    r.z = u32x4{0, 0, 0, 0};
    r.f[0] = r.f[1] = f32x4{0.f, 0.f, 0.f, 0.f};
    r.live = false;
    const int d0 = (z_polar ? 0 : n0) + i.d0;
    if (n.t0 + i.row < seg.len && (z_polar || i.d0 < NT) && d0 < zr.cols) {
      const int row = row_of(n.t0 + i.row);
      r.live = !yz_key || kept(row);
      if (r.live) r.z = lin_load8(zr.p + (int64_t)seg.batch * zr.s[0] + (int64_t)(by_query ? hk : n.hq) * zr.s[1] + (int64_t)row * zr.s[2], d0, zr.cols, zr.vec);
      if (z_polar && c.R) lin_angles8(lin_angle_row(c, seg.batch, row), d0, c.R, c.f_vec, r.f);
    }
    return r;
  };
  // ... and expanded into LDS
  const float* xt = kind == kLinDv ? turns : nullptr;                       // keys carry the bias
  const float* yt = kind == kLinOut ? turns : nullptr;
  const float* zt = kind == kLinDq ? turns : nullptr;
  const float xs = kind == kLinOut ? c.scale : 1.f, ys = kind == kLinDv ? c.scale : 1.f, zs = kind == kLinDk ? c.scale : 1.f;   // queries the scale
  const auto put_xy = [&](const Turn& n, int u, const In& r) {
    const Item i(u);
    if (i.d0 >= xr.cols || i.d0 >= P) return;
    if (xy_polar) {
      if (n.lx) lin_put_polar<T, PL, true>(X, i.row, i.d0, r.x, r.f, r.lx, xs, xt, c.D, c.R, 0, P);
      if (n.lyz) lin_put_polar<T, PL, false>(Y, i.row, i.d0, r.y, r.f, r.ly, ys, yt, c.D, c.R, 0, P);
    } else {
      if (n.lx) lin_put_plain<T, PL, true>(X, i.row, i.d0, r.x);
      if (n.lyz) lin_put_plain<T, PL, false>(Y, i.row, i.d0, r.y);
    }
  };
  const auto put_z = [&](const Turn& n, int u, const InZ& r) {
    const Item i(u);
    if ((!z_polar && i.d0 >= NT) || (z_polar ? 0 : n0) + i.d0 >= zr.cols) return true;
    if (z_polar) return lin_put_polar<T, PL, false>(Z, i.row, i.d0, r.z, r.f, r.live, zs, zt, c.D, c.R, n0, NT);
    return lin_put_plain<T, PL, false>(Z, i.row, i.d0, r.z);
  };
  // Narrow tiles are loaded a chunk ahead, into registers; wide ones, whose state takes those, chunk by chunk.
  constexpr bool kAhead = P <= 128 && NT <= 128;
  In xy[kAhead ? K::TP : 1];
  InZ zz[kAhead ? K::TZ : 1];
  const auto load = [&](int it) {
    if constexpr (kAhead) {
      const Turn n = turn_of(it);
#pragma unroll
      for (int u = 0; u < K::TP; ++u) xy[u] = load_xy(n, u);
      if (n.lyz)
#pragma unroll
        for (int u = 0; u < K::TZ; ++u) zz[u] = load_z(n, u);
    }
  };
  const auto store = [&](int it) {
    const Turn n = turn_of(it);
    bool fin = true;
    if constexpr (kAhead) {
#pragma unroll
      for (int u = 0; u < K::TP; ++u) put_xy(n, u, xy[u]);
      if (n.lyz)
#pragma unroll
        for (int u = 0; u < K::TZ; ++u) fin &= put_z(n, u, zz[u]);
    } else {
      const int txy = (C * ((xr.cols + 31) / 32 * 4) + kThreads - 1) / kThreads;
#pragma unroll 1
      for (int u = 0; u < txy; ++u) put_xy(n, u, load_xy(n, u));
      const int tz = (C * ((min(z_polar ? 256 : NT, zr.cols) + 31) / 32 * 4) + kThreads - 1) / kThreads;
      if (n.lyz)
#pragma unroll 1
        for (int u = 0; u < tz; ++u) fin &= put_z(n, u, load_z(n, u));
    }
    if (!fin) odd[it & 1] = 1;
  };

  f32x4 O[CT][IT];
  const int turns_n = chunks * ng;
  bool odd_z = false;
  load(0);
  for (int it = 0; it < turns_n; ++it) {
    const int ch = it / ng, g = it - ch * ng, t0 = ch * C;
    __syncthreads();   // nothing reads the tiles any more
    store(it);
    if (it + 1 < turns_n) load(it + 1);
    __syncthreads();
    if (!by_query || g == 0) odd_z = odd[it & 1] != 0;
    // x . y of the rows of 16 x 16 tiles j <= i, weighted
    constexpr int kTiles = IT * (IT + 1) / 2;
#pragma unroll 1
    for (int t = wave; t < kTiles; t += K::NW) {
      const int ti = t == 0 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3, tj = t - ti * (ti + 1) / 2;
      f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
      for (int k = 0; k < steps; ++k) {
        u32x4 xa[PL], ya[PL];
#pragma unroll
        for (int l = 0; l < PL; ++l) {
          xa[l] = lin_along_placed(X.p + l * X.plane, K::XS, 16 * ti, 32 * k, lane);
          ya[l] = lin_along(Y.p + l * Y.plane, K::YS, 16 * tj, 32 * k, lane);
        }
        s = lin_mfma<PL, PL>(ya, xa, s);
      }
      const int i = 16 * ti + l16, j0 = 16 * tj + 4 * q4;
      f32x4 w;
#pragma unroll
      for (int r = 0; r < 4; ++r) w[r] = j0 + r <= i ? s[r] * lin_power(lg, i - j0 - r) : 0.f;
      u32x2 wp[PL];
      lin_pack4<PL>(w, wp);
#pragma unroll
      for (int l = 0; l < PL; ++l) *reinterpret_cast<u32x2*>(A.p + l * A.plane + i * K::AS + lin_place<true>(j0)) = wp[l];
    }
    // W^T x
    if (busy && (by_query || g == 0)) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int i = 0; i < IT; ++i) O[ct][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < ST; ++s)
        if (s < steps) {
          u32x4 wa[CT][PL];
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) {
            u32x2 lo[PL], hi[PL];
            lin_pack4<PL>(W[ct][2 * s], lo);
            lin_pack4<PL>(W[ct][2 * s + 1], hi);
#pragma unroll
            for (int l = 0; l < PL; ++l) wa[ct][l] = u32x4{lo[l][0], lo[l][1], hi[l][0], hi[l][1]};
          }
#pragma unroll
          for (int i = 0; i < IT; ++i) {
            u32x4 xa[PL];
#pragma unroll
            for (int l = 0; l < PL; ++l) xa[l] = lin_along_placed(X.p + l * X.plane, K::XS, 16 * i, 32 * s, lane);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) O[ct][i] = lin_mfma<PL, PL>(wa[ct], xa, O[ct][i]);
          }
        }
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const float w = lin_power(lg, 16 * i + l16 + a);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) O[ct][i] *= w;
      }
    }
    __syncthreads();   // the weighted products are there
    if (tid == 0) odd[(it + 1) & 1] = 0;   // of the turn before, which nothing reads any more
    if (busy) {
      u32x4 za[CT][KS][PL];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int l = 0; l < PL; ++l) za[ct][s][l] = lin_across(Z.p + l * Z.plane, K::ZS, 32 * s, col0 + 16 * ct, lane);
      if (!odd_z) {
#pragma unroll
        for (int i = 0; i < IT; ++i)
#pragma unroll
          for (int s = 0; s < KS; ++s)
            if (32 * s <= 16 * i + 15) {
              u32x4 aa[PL];
#pragma unroll
              for (int l = 0; l < PL; ++l) aa[l] = lin_along_placed(A.p + l * A.plane, K::AS, 16 * i, 32 * s, lane);
#pragma unroll
              for (int ct = 0; ct < CT; ++ct) O[ct][i] = lin_mfma<PL, PL>(za[ct][s], aa, O[ct][i]);
            }
      } else {
        // 0 x inf of a row behind would be NaN: rows up to i only
        POPE_COLD_PATH();
#pragma unroll
        for (int i = 0; i < IT; ++i)
#pragma unroll 1
          for (int j = 0; j <= 16 * i + l16; ++j) {
            float w = 0.f;
            for (int l = 0; l < PL; ++l) w += BF16::to_float(A.p[l * A.plane + (16 * i + l16) * K::AS + lin_place<true>(j)]);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                float z = BF16::to_float(Z.p[j * K::ZS + col0 + 16 * ct + 4 * q4 + r]);
                if constexpr (PL == 2)
                  if (fabsf(z) <= 3.402823466e38f) z += BF16::to_float(Z.p[Z.plane + j * K::ZS + col0 + 16 * ct + 4 * q4 + r]);
                O[ct][i][r] += w * z;
              }
          }
      }
      // the next chunk's W
      if (ch + 1 < chunks && (!by_query || g == ng - 1)) {
        if (by_query || g == 0) {
#pragma unroll
          for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int s = 0; s < 2 * ST; ++s) W[ct][s] *= keep;
        }
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            float v[8];
            unpack8<BF16>(za[ct][s][0], v);
            if constexpr (PL == 2) {
              float v2[8];
              unpack8<BF16>(za[ct][s][1], v2);
#pragma unroll
              for (int j = 0; j < 8; ++j) v[j] += v2[j];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] *= wz[s][j];
            u32x2 lo[PL], hi[PL];
            lin_pack4<PL>(f32x4{v[0], v[1], v[2], v[3]}, lo);
            lin_pack4<PL>(f32x4{v[4], v[5], v[6], v[7]}, hi);
#pragma unroll
            for (int l = 0; l < PL; ++l) za[ct][s][l] = u32x4{lo[l][0], lo[l][1], hi[l][0], hi[l][1]};
          }
#pragma unroll
        for (int e = 0; e < 2 * ST; ++e)
          if (e < 2 * steps) {
#pragma unroll
            for (int s = 0; s < KS; ++s) {
              u32x4 ya[PL];
#pragma unroll
              for (int l = 0; l < PL; ++l) ya[l] = lin_across(Y.p + l * Y.plane, K::YS, 32 * s, 16 * e, lane);
#pragma unroll
              for (int ct = 0; ct < CT; ++ct) W[ct][e] = lin_mfma<PL, PL>(ya, za[ct][s], W[ct][e]);
            }
          }
      }
      // out: a lane has row 16 i + l16, columns 4 q4 .. of each tile
      if (by_query || g == ng - 1) {
        const int h = by_query ? (g0 + g) * c.Hk + hk : hk;
        uint16_t* ob = out.p + (int64_t)seg.batch * out.s[0] + (int64_t)h * out.s[1];
#pragma unroll
        for (int i = 0; i < IT; ++i) {
          const int t = t0 + 16 * i + l16;
          if (t >= seg.len) continue;
          const int row = row_of(t);
          uint16_t* orow = ob + (int64_t)row * out.s[2];
          if (!chain) {
            const bool dead = kind == kLinDv && !kept(row);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
              const int d = n0 + col0 + 16 * ct + 4 * q4;
              f32x4 v = O[ct][i];
              if (dead) v = f32x4{0.f, 0.f, 0.f, 0.f};
              if (out.vec && d < out_cols) {
                *reinterpret_cast<u32x2*>(orow + d) = u32x2{T::pack2(v[0], v[1]), T::pack2(v[2], v[3])};
              } else {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                  if (d + r < out_cols) orow[d + r] = T::bits(v[r]);
              }
            }
          } else {
            // chain rule of the polar rows: a lane's columns are two (cosine, sine) pairs, or four other dims
            const LinRows in = kind == kLinDq ? c.q : c.k;
            const uint16_t* xrow = in.p + (int64_t)seg.batch * in.s[0] + (int64_t)h * in.s[1] + (int64_t)row * in.s[2];
            const float* frow = c.R ? lin_angle_row(c, seg.batch, row) : nullptr;
            float* ph = p.dphase[which] ? p.dphase[which] + (((int64_t)seg.batch * (kind == kLinDq ? c.Hq : c.Hk) + h) * c.seqs.N + row) * c.R : nullptr;
            const bool dead = kind == kLinDk && !kept(row);
            const float f = kind == kLinDq ? c.scale : 1.f;
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
              const int e0 = n0 + col0 + 16 * ct + 4 * q4;
#pragma unroll
              for (int pr = 0; pr < 2; ++pr) {
                const int e = e0 + 2 * pr;
                const float dc = dead ? 0.f : O[ct][i][2 * pr] * f, ds = dead ? 0.f : O[ct][i][2 * pr + 1] * f;
                if (e < 2 * c.R) {
                  const int d = e >> 1;
                  const float x = T::to_float(xrow[d]);
                  float sn, cs;
                  sincos_turns(frow[d], kind == kLinDk ? turns[d] : 0.f, &sn, &cs);
                  orow[d] = T::bits(dead ? 0.f : sigmoid_f(x) * (dc * cs + ds * sn));
                  const float dth = dead ? 0.f : softplus_f(x) * (ds * cs - dc * sn);
                  dbsum[ct][pr] += dth;
                  if (ph) ph[d] = dth;
                } else {
                  if (e < c.E) orow[e - c.R] = T::bits(dc);
                  if (e + 1 < c.E) orow[e + 1 - c.R] = T::bits(ds);
                }
              }
            }
          }
        }
      }
    }
  }
  if (kind == kLinDk && p.dbias && busy) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int pr = 0; pr < 2; ++pr) {
        float v = dbsum[ct][pr];
#pragma unroll
        for (int i = 1; i < 16; i *= 2) v += wave_shfl_xor(v, i);
        const int e = n0 + col0 + 16 * ct + 4 * q4 + 2 * pr;
        if (l16 == 0 && e < 2 * c.R) p.dbias[((int64_t)at * c.Hk + hk) * c.R + (e >> 1)] = v;
      }
  }
}

// KIND kLinDq: dq and dk, in one launch.
template <typename T, typename K, int KIND>
__global__ __launch_bounds__(K::kThreads, 1) void linear_out_kernel(LinOutParams p) {
  constexpr int kBytes = K::PL * (K::C * (K::XS + K::YS + K::ZS + K::AS)) * 2 + 256 * 4 + 16;
  __shared__ __attribute__((aligned(16))) char smem[kBytes];
  const int wg = blockIdx.x;
  if constexpr (KIND == kLinDq) {
    if (wg >= p.wgs) {
      lin_out_job<T, K, kLinDk>(p, wg - p.wgs, smem);
      return;
    }
  }
  lin_out_job<T, K, KIND>(p, wg, smem);
}

template <typename T, int KIND>
struct LinOutLaunch {
  template <typename K>
  struct Of {
    static hipError_t go(LinOutParams p, const char* name, hipStream_t s) {
      const LinCall& c = p.c;
      const int64_t segs = c.seqs.T + (c.seqs.cu ? 1 : 0);
      p.tiles = ((KIND == kLinDq ? c.E : c.Dv) + K::NT - 1) / K::NT;
      const int64_t n = segs * p.tiles * c.Hk * (KIND == kLinDv ? 1 : c.G / p.heads_per), all = n + (KIND == kLinDq ? segs * p.tiles * c.Hk : 0);
      if (all >= ((int64_t)1 << 22)) return hipErrorInvalidValue;
      p.wgs = (int)n;
      return launch_named(name, linear_out_kernel<T, K, KIND>, dim3((unsigned)all), dim3(K::kThreads), s, p);
    }
  };
};
template <typename T, int KIND>
hipError_t launch_linear_out_t(const LinOutParams& p, const char* name, hipStream_t s) {
  return lin_dispatch<T, LinOutLaunch<T, KIND>::template Of>(KIND == kLinDq ? p.c.Dv : p.c.E, KIND == kLinDq ? p.c.E : p.c.Dv, p, name, s);
}

}  // namespace pope
