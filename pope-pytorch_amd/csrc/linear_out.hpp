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
// Rounding: x, y, z, the weighted C x C products and W as an operand are bf16: one part for bf16 rows (each is off by at most 2^-8,
// as the output is by its own rounding), the sum of two for fp16 and fp32 rows, for bf16 rows whose output goes on in fp32, and for
// calls of up to 32 bf16 rows (2^-16; C is 32 then).  W itself, all sums and the powers of g are fp32.
//
// What bounds it: waits.  32,768 rows of 8 heads, D 64, R 32, bf16: 45-48 us for the outputs (6.4 GFLOP, 167 MB, 3.5 TB/s); 2 x 4,096 of
// them: outputs 19, dq and dk 62, dv 20.  D 256, R 256 (2 x 2,048 rows): 80, 213 and 80, where a segment's state is 512 KB, its load a
// burst of 15 us, and one workgroup has a CU.  A chunk's tiles come a chunk ahead where registers allow; two workgroups a CU cover for
// each other where LDS allows.
#pragma once
#include <algorithm>
#include <type_traits>

#include "linear_dev.hpp"

namespace pope {

template <bool B>
using Bool = std::integral_constant<bool, B>;

template <typename K, int KIND>
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

  // packed calls have a workgroup more than there can be segments
  const LinSeg seg = lin_segment(c.seqs, c.seqs.cu && at == c.seqs.T ? kLinNone : at);
  if (seg.seq < 0) {
    if (kind == kLinDk && p.dbias && at < c.seqs.T)
      for (int d = tid; d < c.R; d += kThreads) p.dbias[((int64_t)at * c.Hk + hk) * c.R + d] = 0.f;
    // Rows outside every sequence become zeros, a row a wave, by all workgroups without a segment (200 rows in a buffer of 32,768, 8
    // heads, D 64, bf16: one workgroup a head took 1,879 us for the call, all of them 71).
    const int total = (unsigned)seg.m < (unsigned)c.seqs.T ? seg.m : c.seqs.T;   // bounds that descend may have any
    const int workers = (c.seqs.T + 1 - total) * tiles, worker = (at - total) * tiles + tile;
    const int lo = lin_bound(c.seqs, 0), hi = lin_bound(c.seqs, c.seqs.B);
    for (int64_t r = worker * K::NW + wave; r < lo + c.seqs.N - hi; r += workers * K::NW) {
      const int64_t row = r < lo ? r : hi + r - lo;
      for (int g = 0; g < (by_query ? ng : 1); ++g) {
        const int h = by_query ? (g0 + g) * c.Hk + hk : hk;
        lin_set4<PL>(out, lin_base(out, 0, h, row), 0u, 4 * lane, f32x4{0.f, 0.f, 0.f, 0.f});
        if (chain && p.dphase[which])
          for (int d = lane; d < c.R; d += 64) p.dphase[which][((int64_t)h * c.seqs.N + row) * c.R + d] = 0.f;
      }
    }
    return;
  }

  uint16_t* lds = reinterpret_cast<uint16_t*>(smem);
  const LinTile X{lds, K::XS, C * K::XS};
  const LinTile Y{X.p + PL * X.plane, K::YS, C * K::YS};
  const LinTile Z{Y.p + PL * Y.plane, K::ZS, C * K::ZS};
  const LinTile A{Z.p + PL * Z.plane, K::AS, C * K::AS};
  float* later = reinterpret_cast<float*>(A.p + PL * A.plane);   // C: weights of a chunk's rows in the next state
  float* turns = later + C;                                      // kLinDk: 256
  int* odd = reinterpret_cast<int*>(turns + (chain ? 256 : 0));   // z of this chunk that are not finite; two, by turns
  const float lg = lin_log2(c, hk);
  const int a = rev ? 0 : 1;
  const int chunks = (seg.len + C - 1) / C;
  // The wave's columns in the tile: 16 and, where it has two tiles, 16 half of the tile further on, so that the rotated columns, which
  // come first and take the chain rule, fall to all waves (dq and dk of 16 heads on 4, 128 + 64 columns: 112 us with 32 columns in a row, 109 so).
  constexpr int kStep = 16 * K::NW;
  const int col0 = 16 * wave;
  const bool busy = n0 + col0 < ncols;
  const int steps = (pcols + 31) / 32;

  float dbsum[CT][2];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) dbsum[ct][0] = dbsum[ct][1] = 0.f;

  // Rows of a chunk, t of 0 .. C - 1 in the job's order, from the chunk's base row on.
  const auto base_row = [&](int t0) { return (int64_t)seg.row0 + (rev ? seg.len - C - t0 : t0); };   // reverse: may be in front of the first row
  const auto place = [&](int t) { return (uint32_t)(rev ? C - 1 - t : t); };
  typedef LinItem<C, kThreads> Item;
  // The thread's number as something new in every turn: places in memory and LDS are worked out again where they are used, instead of
  // held in registers for the whole loop (the compiler did, and spilled the state for it).
  int tv = tid;
  // x, y and z are expanded rows or plain ones, the keys' and values' rows among the latter, which the mask may leave out
  constexpr bool x_hat = !chain, y_hat = !chain, z_hat = chain;
  const LinRows xr = kind == kLinDq ? c.g : c.v, yr = kind == kLinDq ? c.v : c.g, zr = kind == kLinOut ? c.v : c.g;
  const LinHat xh = kind == kLinOut ? c.qh : c.kh, yh = kind == kLinOut ? c.kh : c.qh, zh = kind == kLinDq ? c.kh : c.qh;
  constexpr bool x_key = kind == kLinDk, y_key = kind == kLinDq, z_key = kind == kLinOut;
  const int xcols = x_hat ? xh.EP : xr.cols, ycols = y_hat ? yh.EP : yr.cols, zcols = z_hat ? zh.EP : zr.cols;   // x and y have as many
  struct Turn { int t0, hq; bool lx, lyz; };
  const auto turn_of = [&](int it) {
    const int ch = it / ng, g = it - ch * ng;
    return Turn{ch * C, (g0 + g) * c.Hk + hk, by_query || g == 0, !by_query || g == 0};
  };
  // Loads keep what they read as it is until it is put, and nothing decides whether they happen: a conversion, a choice by a mask's
  // byte or a branch around a load would wait for it.  Rows behind the segment are the last one's again, and what they and the mask's
  // rows gave becomes zeros on the way into LDS.  Plain rows that are not whole 16-byte units take another way, branches and all.
  const uint8_t* mask = c.mask ? c.mask + (int64_t)seg.batch * c.mask_sb : nullptr;
  const auto mask_base = [&](int t0) { return mask ? reinterpret_cast<const uint8_t*>(lin_uniform(mask + base_row(t0))) : nullptr; };
  const auto kept = [&](const uint8_t* m, int t) { return m ? (uint32_t)m[place(t)] : 1u; };
  // A thread's chunks of the tiles, read from memory.
  struct Part { LinRaw<PL> w; uint32_t keep; };
  const auto base_of = [&](auto hat, const LinHat& t, const LinRows& r, int h, int t0) {
    if constexpr (decltype(hat)::value) return lin_uniform(t.p + (((int64_t)seg.batch * t.H + h) * c.seqs.N + base_row(t0)) * t.EP);
    else return lin_base(r, seg.batch, h, base_row(t0));
  };
  const auto get = [&](auto hat, auto key, auto whole, const LinHat& t, const LinRows& r, const char* base, const uint8_t* m, int cols, int t0, const Item& i, int d0) {
    Part o;
    const int at = min(i.row, seg.len - 1 - t0);
    d0 = min(d0, (cols - 1) & ~7);
    if constexpr (decltype(hat)::value) {
      const uint32_t off = (place(at) * t.EP + d0) * 2;
      o.w.a = *reinterpret_cast<const u32x4*>(base + off);
      if constexpr (PL == kTwo) o.w.b = *reinterpret_cast<const u32x4*>(base + 2 * t.plane + off);
    } else {
      o.w = lin_load8<PL>(r, base, place(at) * lin_step(r), d0, decltype(whole)::value);
    }
    if constexpr (decltype(key)::value) o.keep = kept(m, at);
    return o;
  };
  struct Bases { const char *x, *y, *z; const uint8_t* m; };
  const auto bases_of = [&](const Turn& n) {
    return Bases{base_of(Bool<x_hat>{}, xh, xr, by_query ? n.hq : hk, n.t0), base_of(Bool<y_hat>{}, yh, yr, by_query ? hk : n.hq, n.t0),
                 base_of(Bool<z_hat>{}, zh, zr, by_query ? hk : n.hq, n.t0), mask_base(n.t0)};
  };
  const auto get_x = [&](auto whole, const Turn& n, const Bases& b, int u) {
    const Item i(u, tv);
    return get(Bool<x_hat>{}, Bool<x_key>{}, whole, xh, xr, b.x, b.m, xcols, n.t0, i, i.d0);
  };
  const auto get_y = [&](auto whole, const Turn& n, const Bases& b, int u) {
    const Item i(u, tv);
    return get(Bool<y_hat>{}, Bool<y_key>{}, whole, yh, yr, b.y, b.m, ycols, n.t0, i, i.d0);
  };
  const auto get_z = [&](auto whole, const Turn& n, const Bases& b, int u) {
    const Item i(u, tv);
    return get(Bool<z_hat>{}, Bool<z_key>{}, whole, zh, zr, b.z, b.m, zcols, n.t0, i, n0 + i.d0);
  };
  // ... and put into LDS
  const auto put = [&](auto hat, auto key, auto perm, const LinRows& r, const LinTile& t, int t0, const Item& i, Part o) {
    constexpr bool kPerm = decltype(perm)::value;
    if (t0 + i.row >= seg.len || (decltype(key)::value && !o.keep)) o.w = LinRaw<PL>{};
    if constexpr (!decltype(hat)::value) {
      return lin_put_plain<PL, kPerm>(t, i.row, i.d0, o.w, r.type);
    } else {
      if constexpr (PL == kTwo) {
        const u32x4 both[2] = {o.w.a, o.w.b};
        lin_put_parts<2, kPerm>(t, i.row, i.d0, both);
      } else {
        lin_put_parts<1, kPerm>(t, i.row, i.d0, &o.w.a);
      }
      return lin_odd8(o.w.a);
    }
  };
  const auto put_x = [&](const Turn& n, int u, const Part& o) {
    const Item i(u, tv);
    if (i.d0 < xcols) put(Bool<x_hat>{}, Bool<x_key>{}, Bool<true>{}, xr, X, n.t0, i, o);
  };
  const auto put_y = [&](const Turn& n, int u, const Part& o) {
    const Item i(u, tv);
    if (i.d0 < ycols) put(Bool<y_hat>{}, Bool<y_key>{}, Bool<false>{}, yr, Y, n.t0, i, o);
  };
  const auto put_z = [&](const Turn& n, int u, const Part& o) {
    const Item i(u, tv);
    return i.d0 < NT && n0 + i.d0 < zcols && put(Bool<z_hat>{}, Bool<z_key>{}, Bool<false>{}, zr, Z, n.t0, i, o);
  };
  const bool whole_rows = (x_hat || xr.vec) && (y_hat || yr.vec) && (z_hat || zr.vec);
  // Narrow tiles are loaded a chunk ahead, into registers; wide ones, whose state takes those, when the chunk's turn
  // begins: x and z at once, then y in the registers that these leave; where eight waves have a chain's wide state, two at a time (dq and
  // dk of 256 columns: 222 us against 194).
  constexpr bool kAhead = P <= 128 && NT <= 128;
  constexpr bool kFew = chain && P > 128 && K::NW == 8;
  constexpr int kTX = K::TP, kTZ = K::TZ;
  Part xin[kTX], yin[kTX], zin[kTZ];
  const auto load_as = [&](auto whole, int it, bool xz, bool y) {
    const Turn n = turn_of(it);
    const Bases b = bases_of(n);
    if (xz && n.lx)
#pragma unroll
      for (int u = 0; u < kTX; ++u) xin[u] = get_x(whole, n, b, u);
    if (xz && n.lyz)
#pragma unroll
      for (int u = 0; u < kTZ; ++u) zin[u] = get_z(whole, n, b, u);
    if (y && n.lyz)
#pragma unroll
      for (int u = 0; u < kTX; ++u) yin[u] = get_y(whole, n, b, u);
  };
  const auto load = [&](int it, bool xz, bool y) {
    if (whole_rows) load_as(Bool<true>{}, it, xz, y);
    else load_as(Bool<false>{}, it, xz, y);
  };
  const auto turns_for = [&](int cols) { return (C * ((cols + 31) / 32 * 4) + kThreads - 1) / kThreads; };
  const auto store_few = [&](auto whole, const Turn& n) {
    const Bases b = bases_of(n);
    bool some = false;
    const int txy = turns_for(xcols);
#pragma unroll 2
    for (int u = 0; u < txy; ++u) {
      Part x, y;
      if (n.lx) x = get_x(whole, n, b, u);
      if (n.lyz) y = get_y(whole, n, b, u);
      if (n.lx) put_x(n, u, x);
      if (n.lyz) put_y(n, u, y);
    }
    if (n.lyz) {
      const int tz = turns_for(min(NT, zcols - n0));
#pragma unroll 4
      for (int u = 0; u < tz; ++u) some |= put_z(n, u, get_z(whole, n, b, u));
    }
    return some;
  };
  const auto store = [&](int it) {
    const Turn n = turn_of(it);
    bool some = false;
    if constexpr (kFew) {
      some = whole_rows ? store_few(Bool<true>{}, n) : store_few(Bool<false>{}, n);
      if (some) odd[it & 1] = 1;
      return;
    }
    if (n.lx)
#pragma unroll
      for (int u = 0; u < kTX; ++u) put_x(n, u, xin[u]);
    if (n.lyz)
#pragma unroll
      for (int u = 0; u < kTZ; ++u) some |= put_z(n, u, zin[u]);
    if constexpr (!kAhead) load(it, false, true);
    if (n.lyz)
#pragma unroll
      for (int u = 0; u < kTX; ++u) put_y(n, u, yin[u]);
    if (some) odd[it & 1] = 1;
  };

  // A row alone: the norm behind it leaves of its gradient what is at right angles to the row itself, so dO . v is a sum that all but
  // cancels, 500 times and more.  Its sum is over fp32 values then, not their parts; it goes on as two parts, as the row that it multiplies.
  const bool lone = PL == kTwo && seg.len == 1;
  f32x4 O[CT][IT];
  const int turns_n = chunks * ng;
  bool odd_z = false;
  if constexpr (kAhead) load(0, true, true);
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
      const bool whole = chain && c.Dv % 4 == 0 && (reinterpret_cast<uintptr_t>(from) & 15) == 0;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        const int col = n0 + col0 + kStep * ct + l16;
#pragma unroll
        for (int s = 0; s < 2 * ST; ++s) {
          const int row = 16 * s + 4 * q4;
          if (whole) {   // transposed where the result has expanded columns
            if (row < pcols && col < ncols) W[ct][s] = *reinterpret_cast<const f32x4*>(from + (int64_t)col * c.Dv + row);
            continue;
          }
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (row + r < pcols && col < ncols) W[ct][s][r] = chain ? from[(int64_t)col * c.Dv + row + r] : from[(int64_t)(row + r) * c.Dv + col];
        }
      }
    }
  }
  const float keep = lin_power(lg, C);
  for (int t = tid; t < C; t += kThreads) later[t] = lin_power(lg, C - a - t);
  constexpr int kTileBytes = PL * (C * (K::XS + K::YS + K::ZS + K::AS)) * 2;
  for (int i = tid; i < kTileBytes / 16; i += kThreads) reinterpret_cast<u32x4*>(smem)[i] = u32x4{0, 0, 0, 0};
  if (tid < 2) odd[tid] = 0;
  if (kind == kLinDk)
    for (int d = tid; d < c.R; d += kThreads) turns[d] = lin_turns(lin_bias(c, hk, d));

  for (int it = 0; it < turns_n; ++it) {
    const int ch = it / ng, g = it - ch * ng, t0 = ch * C;
    // places are worked out anew each turn: kept across turns, they leave the chains and the two-part products no registers (dq and
    // dk of 256 columns: 399 us with spills, 194 without), nor wide states and outputs with two tiles a wave; the others have the room, and save 5 to 8 us in 70
    if constexpr (chain || PL == kTwo || CT > 1 || P > 128) tv = (int)opaque_u32((uint32_t)tid);
    const int lane = tv & 63, q4 = lane >> 4, l16 = lane & 15;
    if constexpr (!kAhead && !kFew) load(it, true, false);
    __syncthreads();   // nothing reads the tiles any more
    store(it);
    if (kAhead && it + 1 < turns_n) load(it + 1, true, true);
    __syncthreads();
    if (!by_query || g == 0) odd_z = odd[it & 1] != 0 || lone;
    // x . y of the rows of 16 x 16 tiles j <= i, weighted: a wave has tiles of one i
    {
      constexpr int kShare = K::NW / IT, kTiles = IT > kShare ? IT / kShare : 1;
      const int ti = wave / kShare, j0 = wave % kShare;
      f32x4 sc[kTiles];
#pragma unroll
      for (int j = 0; j < kTiles; ++j) sc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < ST; ++k)
        if (k < steps) {
          u32x4 xa[PL], ya[kTiles][PL];
#pragma unroll
          for (int l = 0; l < PL; ++l) {
            xa[l] = lin_along_placed(X.p + l * X.plane, K::XS, 16 * ti, 32 * k, lane);
#pragma unroll
            for (int j = 0; j < kTiles; ++j)
              if (j0 + j * kShare <= ti) ya[j][l] = lin_along(Y.p + l * Y.plane, K::YS, 16 * (j0 + j * kShare), 32 * k, lane);
          }
#pragma unroll
          for (int j = 0; j < kTiles; ++j)
            if (j0 + j * kShare <= ti) sc[j] = lin_mfma<PL, PL>(ya[j], xa, sc[j]);
        }
      if (chain && lone && wave == 0) {
        const int64_t row = base_row(0) + place(0);
        const int hq = turn_of(it).hq;
        float dot = 0.f;
        for (int d = lane; d < c.Dv; d += 64)
          dot += lin_get<PL>(c.g, seg.batch * c.g.s[0] + hq * c.g.s[1] + row * c.g.s[2] + d) * lin_get<PL>(c.v, seg.batch * c.v.s[0] + hk * c.v.s[1] + row * c.v.s[2] + d);
#pragma unroll
        for (int m = 1; m < 64; m *= 2) dot += wave_shfl_xor(dot, m);
        if (lane == 0) sc[0][0] = kept(mask_base(0), 0) ? dot : 0.f;
      }
#pragma unroll
      for (int j = 0; j < kTiles; ++j) {
        if (j0 + j * kShare > ti) continue;
        const int i = 16 * ti + l16, jr = 16 * (j0 + j * kShare) + 4 * q4;
        f32x4 w;
#pragma unroll
        for (int r = 0; r < 4; ++r) w[r] = jr + r <= i ? sc[j][r] * lin_power(lg, i - jr - r) : 0.f;
        u32x2 wp[PL];
        lin_pack4<PL>(w, wp);
#pragma unroll
        for (int l = 0; l < PL; ++l) *reinterpret_cast<u32x2*>(A.p + l * A.plane + i * K::AS + lin_place<true>(jr)) = wp[l];
      }
    }
    // what the chain rule of this turn's rows reads, ahead: a lane has row 16 i + l16, and, of each 16 columns, two dims
    const bool ends = by_query || g == ng - 1;
    const bool pairs = out.vec && (kind == kLinDq ? c.q : c.k).vec && (c.f_vec || !c.R);   // two dims at a time: R, D multiples of 8
    LinPair<PL> cx[CT][IT];
    f32x2 cf[CT][IT];
    uint32_t live[IT];
    const int h_out = by_query ? (g0 + g) * c.Hk + hk : hk;
    if constexpr (rev) {
      const uint8_t* m = mask_base(t0);
#pragma unroll
      for (int i = 0; i < IT; ++i) live[i] = kept(m, min(16 * i + l16, seg.len - 1 - t0));
    }
    const LinRows in = kind == kLinDq ? c.q : c.k;   // chain
    const char* in_base = chain ? lin_base(in, seg.batch, h_out, base_row(t0)) : nullptr;
    const char* f_base = chain && c.R ? lin_uniform(c.freqs + (int64_t)seg.batch * c.f_s[0] + base_row(t0) * c.f_s[1]) : nullptr;
    if constexpr (chain) {
      if (pairs && c.R) {
#pragma unroll
        for (int i = 0; i < IT; ++i) {
          const uint32_t at = place(min(16 * i + l16, seg.len - 1 - t0));
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) {
            const int d = min((n0 + col0 + kStep * ct + 4 * q4) >> 1, c.R - 2);
            cx[ct][i] = lin_get2<PL>(in, in_base, at * lin_step(in), d);
            cf[ct][i] = *reinterpret_cast<const f32x2*>(f_base + (at * (uint32_t)c.f_s[1] + d) * 4);
          }
        }
      }
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
          for (int l = 0; l < PL; ++l) za[ct][s][l] = lin_across(Z.p + l * Z.plane, K::ZS, 32 * s, col0 + kStep * ct, lane);
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
          for (int j = 0; j <= 16 * i + l16 && !(lone && j); ++j) {
            float w = 0.f;
            for (int l = 0; l < PL; ++l) w += BF16::to_float(A.p[l * A.plane + (16 * i + l16) * K::AS + lin_place<true>(j)]);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                float z = BF16::to_float(Z.p[j * K::ZS + col0 + kStep * ct + 4 * q4 + r]);
                if constexpr (PL == 2)
                  if (fabsf(z) <= kF32Max) z += BF16::to_float(Z.p[Z.plane + j * K::ZS + col0 + kStep * ct + 4 * q4 + r]);
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
            const f32x4 w0 = *reinterpret_cast<const f32x4*>(later + 32 * s + 4 * q4), w1 = *reinterpret_cast<const f32x4*>(later + 32 * s + 16 + 4 * q4);
            float v[8];
            unpack8<BF16>(za[ct][s][0], v);
            if constexpr (PL == 2) {
              float v2[8];
              unpack8<BF16>(za[ct][s][1], v2);
#pragma unroll
              for (int j = 0; j < 8; ++j) v[j] += v2[j];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] *= w0[j], v[4 + j] *= w1[j];
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
      if (ends) {
        char* ob = lin_base(out, seg.batch, h_out, base_row(t0));
        float* phase = nullptr;
        if constexpr (chain)
          if (p.dphase[which]) phase = p.dphase[which] + (((int64_t)seg.batch * (kind == kLinDq ? c.Hq : c.Hk) + h_out) * c.seqs.N + base_row(t0)) * c.R;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
          const int t = 16 * i + l16;
          if (t0 + t >= seg.len) continue;
          const uint32_t orow = place(t) * lin_step(out);
          if (!chain) {
            const bool dead = rev && !live[i];
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
              lin_set4<PL>(out, ob, orow, n0 + col0 + kStep * ct + 4 * q4, dead ? f32x4{0.f, 0.f, 0.f, 0.f} : O[ct][i]);
          } else {
            // chain rule of the polar rows: a lane's columns are two (cosine, sine) pairs, or four other dims
            const bool dead = rev && !live[i];
            const float f = kind == kLinDq ? c.scale : 1.f;
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
              const int e0 = n0 + col0 + kStep * ct + 4 * q4;
              f32x4 v = O[ct][i] * f;
              if (dead) v = f32x4{0.f, 0.f, 0.f, 0.f};
              float dx[2], x2[2];
              f32x2 f2 = cf[ct][i];
              if (pairs) {
                lin_unpack2<PL>(cx[ct][i], in.type, x2);
              } else {
#pragma unroll
                for (int pr = 0; pr < 2; ++pr) {
                  const int d = min((e0 >> 1) + pr, c.R - 1);
                  x2[pr] = c.R ? lin_get1<PL>(in, in_base, place(t) * lin_step(in), d) : 0.f;
                  f2[pr] = c.R ? *reinterpret_cast<const float*>(f_base + (place(t) * (uint32_t)c.f_s[1] + d) * 4) : 0.f;
                }
              }
#pragma unroll
              for (int pr = 0; pr < 2; ++pr) {
                const int e = e0 + 2 * pr;
                const float dc = v[2 * pr], ds = v[2 * pr + 1];
                if (e < 2 * c.R) {
                  const int d = e >> 1;
                  const float x = x2[pr];
                  float sn, cs;
                  sincos_turns(f2[pr], kind == kLinDk ? turns[d] : 0.f, &sn, &cs);
                  float soft, slope;
                  lin_soft(x, &soft, &slope);
                  dx[pr] = dead ? 0.f : slope * (dc * cs + ds * sn);
                  const float dth = dead ? 0.f : soft * (ds * cs - dc * sn);
                  dbsum[ct][pr] += dth;
                  if (phase) phase[place(t) * c.R + d] = dth;
                  if (!pairs) lin_put_value<PL>(out, ob, orow, d, dx[pr]);
                } else if (!pairs) {
                  if (e < c.E) lin_put_value<PL>(out, ob, orow, e - c.R, dc);
                  if (e + 1 < c.E) lin_put_value<PL>(out, ob, orow, e + 1 - c.R, ds);
                }
              }
              if (pairs) {
                if (e0 < 2 * c.R) lin_set2<PL>(out, ob, orow, e0 >> 1, dx[0], dx[1]);
                else if (e0 < c.E) lin_set4<PL>(out, ob, orow, e0 - c.R, v);
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
        const int e = n0 + col0 + kStep * ct + 4 * q4 + 2 * pr;
        if (l16 == 0 && e < 2 * c.R) p.dbias[((int64_t)at * c.Hk + hk) * c.R + (e >> 1)] = v;
      }
  }
}

// LDS of a workgroup, and the waves for a SIMD that registers are cut to: what LDS holds of two workgroups (160 KB for a CU).
template <typename K, int KIND>
constexpr int lin_out_bytes() { return K::PL * (K::C * (K::XS + K::YS + K::ZS + K::AS)) * 2 + (K::C + (KIND == kLinDq ? 256 : 0)) * 4 + 16; }
template <typename K, int KIND>
constexpr int lin_out_waves() {
  if (2 * lin_out_bytes<K, KIND>() > 160 * 1024) return (K::NW + 3) / 4;
  return 2;
}

// KIND kLinDq: dk and dq, in one launch; dk first, whose workgroups take all query heads of a key head and so the longest.
template <typename K, int KIND>
__global__ __launch_bounds__(K::kThreads, (lin_out_waves<K, KIND>())) void linear_out_kernel(LinOutParams p) {
  constexpr int kBytes = lin_out_bytes<K, KIND>();
  __shared__ __attribute__((aligned(16))) char smem[kBytes];
  const int wg = blockIdx.x;
  if constexpr (KIND == kLinDq) {
    if (wg < p.first_wgs) {
      lin_out_job<K, kLinDk>(p, wg, smem);
      return;
    }
  }
  lin_out_job<K, KIND>(p, wg - p.first_wgs, smem);
}

template <int KIND>
struct LinOutLaunch {
  template <typename K>
  struct Of {
    static hipError_t go(LinOutParams p, const char* name, hipStream_t s) {
      const LinCall& c = p.c;
      const int64_t segs = c.seqs.T + (c.seqs.cu ? 1 : 0);
      p.tiles = ((KIND == kLinDq ? c.E : c.Dv) + K::NT - 1) / K::NT;
      const int64_t n = segs * p.tiles * c.Hk, first = KIND == kLinDq ? n : 0, all = first + n * (KIND == kLinDv ? 1 : c.G / p.heads_per);
      if (all >= ((int64_t)1 << 22)) return hipErrorInvalidValue;
      p.first_wgs = (int)first;
      return launch_named(name, linear_out_kernel<K, KIND>, dim3((unsigned)all), dim3(K::kThreads), s, p);
    }
  };
};
template <int PL, int KIND>
hipError_t launch_linear_out_t(const LinOutParams& p, const char* name, hipStream_t s) {
  return lin_dispatch<PL, LinOutLaunch<KIND>::template Of>(KIND == kLinDq ? p.c.Dv : p.c.E, KIND == kLinDq ? p.c.E : p.c.Dv, p, name, s);
}

}  // namespace pope
