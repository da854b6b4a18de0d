// Attention of new tokens over the paged cache (gfx950): one kernel for single tokens and for chunks.
//
//   o_i = sum_j 2^(s_ij - m_i) v_j / sum_j 2^(s_ij - m_i),   s_ij = scale log2 e  Q_hat_i . K_hat_j,
// j < L, or j <= the row's position (causal).  K_hat rows come expanded from the cache, so there is no transform in the
// loop; Q_hat = [softplus(q) cos F, softplus(q) sin F, q] is computed once per tile.
//
// Rows.  A key head's rows are (new token i, query head of its group g), r = i G + g: grouped heads fill the 16 columns
// of an MFMA that one query head would leave empty, and a tile's rows stand at neighbouring positions.
// Products are transposed: S^T = K_hat Q_hat^T (A = keys), O^T = V^T P^T (A = columns of V).  A lane then has four keys
// of one row of P per 16-key tile, which are, in that order, its k elements of the second product: P goes from one
// MFMA to the next in registers, and since pages hold K and V in operand order (paged_index.hpp) nothing in the loop
// passes through LDS.  Row sums and maxima of a row lie in the four lanes l % 16.
//
// WK waves share a tile's rows and take every WK-th block of 32 keys (few rows: bound by HBM, waves only add loads in
// flight); 4 / WK groups of waves have rows of their own (many rows).  Where the tiles leave the chip idle, `splits`
// workgroups take parts of the key axis and a second launch joins them.
//
// Precision: S, the maxima, sums and O in fp32.  Q_hat is split into the sum of two 16-bit parts (twice the S products:
// rounded once, its error would appear in every score, about 0.4 of an output's own rounding); P is rounded to 16 bits
// once (its errors are independent from key to key).
#pragma once
#include "paged_rows.hpp"

namespace pope {

template <int KS, int VT, int NQ, int WK>
struct PagedShared {
  static constexpr int QST = KS * 32 + 8;   // 16-bit row stride: an odd number of 16-byte units mod 16
  static constexpr int kGroups = 4 / WK;
  static constexpr int kQ = kGroups * 2 * 16 * QST * 2;                      // hi and lo rows of 16 rows per group
  static constexpr int kJoin = WK > 1 ? kGroups * (WK / 2) * NQ * (VT + 1) * 64 * 16 : 0;
  static constexpr int kBytes = kQ > kJoin ? kQ : kJoin;
};

template <typename T, bool Q8, int KS, int VT, int NQ, int WK>
__global__ __launch_bounds__(256) void paged_attn_kernel(PagedAttnParams p) {
  using Sh = PagedShared<KS, VT, NQ, WK>;
  constexpr int kGroups = Sh::kGroups, QST = Sh::QST, kRows = 16 * NQ * kGroups;
  __shared__ __attribute__((aligned(16))) char smem[Sh::kBytes];
  const PagedCache& c = p.c;
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int group = wave / WK, wk = wave % WK;
  const int col = lane & 15, quad = lane >> 4;

  const PagedJob job = paged_job(p);
  const int tile = job.tile, hk = job.hk, split = job.split;
  const PagedTile t = paged_tile(c.seqs, tile, p.G.d, kRows, 1);
  const PagedSeg& g = t.seg;
  const int rows_all = g.n * (int)p.G.d, r0 = t.local * kRows;
  if (r0 >= rows_all) return;
  const bool causal = p.causal != 0;
  const int blocks = paged_tile_blocks(g, t.local, kRows, p.G, causal);
  const PagedRange range = paged_range(blocks, p.splits, p.least, WK, split);
  if (split > 0 && range.begin >= range.end) return;   // the join knows which splits have blocks
  const bool part = paged_parts(blocks, p.splits, p.least, WK) > 1;

  // ---- the lane's rows: column col of each of the wave's NQ column tiles -------------------------------------
  const PagedRowMap map(r0, p.G);
  const int count = min(rows_all - r0, kRows), wx0 = group * 16 * NQ;
  int row_i[NQ], row_h[NQ], lim[NQ];
  bool live[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int x = wx0 + n * 16 + col;
    live[n] = x < count;
    row_i[n] = live[n] ? map.token(x) : 0;
    row_h[n] = live[n] ? map.group(x) * c.Hk + hk : hk;
    lim[n] = live[n] ? paged_limit(g.first + row_i[n], g.len, causal) : 0;
  }
  // keys every live row of the wave sees
  const int least_lim = wx0 < count ? paged_limit(g.first + map.token(wx0), g.len, causal) : 0;

  // ---- Q_hat of the group's rows, 16 at a time, through LDS --------------------------------------------------
  uint16_t* qhi = reinterpret_cast<uint16_t*>(smem) + group * 2 * 16 * QST;
  uint16_t* qlo = qhi + 16 * QST;
  typename T::vec8 qh[NQ][KS], ql[NQ][KS];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    if (n) __syncthreads();
    const int at = wk * 64 + lane;
    for (int it = at; it < 32 * VT; it += 64 * WK)
      paged_query_make<T>(p, paged_query_load<T>(p, g, map, wx0 + n * 16 + it % 16, count, hk, it / 16 * 8), it % 16, it / 16 * 8, QST, qhi, qlo);
    paged_query_tail<16>(p, at, 64 * WK, KS * 32, QST, qhi, qlo);
    __syncthreads();
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qh[n][ks] = as_vec8<typename T::vec8>(*reinterpret_cast<const u32x4*>(qhi + col * QST + ks * 32 + quad * 8));
      ql[n][ks] = as_vec8<typename T::vec8>(*reinterpret_cast<const u32x4*>(qlo + col * QST + ks * 32 + quad * 8));
    }
  }

  // ---- the loop over the wave's blocks -----------------------------------------------------------------------
  constexpr int kKL = Q8 ? KS : 2 * KS, kVL = Q8 ? VT / 2 : VT;   // 16-byte loads per lane and block
  f32x4 acc[NQ][VT];
  float m[NQ], l[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    m[n] = -INFINITY;
    l[n] = 0.f;
#pragma unroll
    for (int v = 0; v < VT; ++v) acc[n][v] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // page numbers of 64 pages at a time, one per lane; one outside the cache becomes -1
  int page_base = 0, pids = 0;
  auto refill = [&](int pg) {
    page_base = pg;
    const int cols = c.seqs.capacity >> (c.blk_shift + 5);
    const int id = c.table[(int64_t)g.b * c.table_sb + min(pg + lane, cols - 1)];
    pids = (unsigned)id < (unsigned)c.pages ? id : -1;
  };
  auto page_of = [&](int blk) {
    const int pg = blk >> c.blk_shift;
    if (pg - page_base >= 64) refill(pg);
    return __builtin_amdgcn_readlane(pids, pg - page_base);
  };
  u32x4 kf[kKL], vf[kVL];
  u32x2 sc[2], sv[2];   // exponent bytes (8-bit caches): [K0..3][V0..3] of the lane's keys of either half
  // operands of a block; loads of pages outside the cache read page 0 and are masked
  auto load_k = [&](int page, int blk) {
    const int pg = max(page, 0);
    constexpr int kB = Q8 ? 1 : 2;
    const char* base = static_cast<const char*>(c.k) + paged_block_off(c, pg, hk, blk, c.k_head, KS * 1024) * kB + lane * 16;
#pragma unroll
    for (int i = 0; i < kKL; ++i) kf[i] = *reinterpret_cast<const u32x4*>(base + i * 1024);
    if constexpr (Q8) {
      const uint8_t* s = c.scales + paged_scale_base(c, pg, hk, blk) + quad * 8;
      sc[0] = *reinterpret_cast<const u32x2*>(s);
      sc[1] = *reinterpret_cast<const u32x2*>(s + 32);
    }
  };
  auto load_v = [&](int page, int blk) {
    const int pg = max(page, 0);
    constexpr int kB = Q8 ? 1 : 2;
    const char* base = static_cast<const char*>(c.v) + paged_block_off(c, pg, hk, blk, c.v_head, VT * 512) * kB + lane * 16;
#pragma unroll
    for (int i = 0; i < kVL; ++i) vf[i] = *reinterpret_cast<const u32x4*>(base + i * 1024);
  };

  int blk = range.begin + wk;
  int page = -1;
  if (blk < range.end) {
    refill(blk >> c.blk_shift);
    page = page_of(blk);
    load_k(page, blk);
    load_v(page, blk);
  }
  for (; blk < range.end; blk += WK) {
    const int next = blk + WK < range.end ? blk + WK : blk;   // the last one is loaded again, unused
    const int next_page = page_of(next);

    // S^T of the block's two key halves
    f32x4 s[NQ][2];
#pragma unroll
    for (int n = 0; n < NQ; ++n) s[n][0] = s[n][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        typename T::vec8 a;
        if constexpr (Q8) a = as_vec8<typename T::vec8>(unpack_e4m3<T>(u32x2{kf[ks][2 * half], kf[ks][2 * half + 1]}, 1.f));
        else a = as_vec8<typename T::vec8>(kf[2 * ks + half]);
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          s[n][half] = T::mfma16(a, qh[n][ks], s[n][half]);
          s[n][half] = T::mfma16(a, ql[n][ks], s[n][half]);
        }
      }
    }
    if constexpr (Q8) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        sv[half] = sc[half];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int e = (int)((sc[half][0] >> (8 * i)) & 0xff) - 127;
#pragma unroll
          for (int n = 0; n < NQ; ++n) s[n][half][i] = __builtin_amdgcn_ldexpf(s[n][half][i], e);
        }
      }
    }
    if (T::kCode == 1 && p.late != 1.f) {
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int half = 0; half < 2; ++half) s[n][half] *= p.late;
    }
    load_k(next_page, next);

    const int key0 = blk * kBlockKeys + quad * 4;   // the lane's keys: key0 + 16 half + i
    const bool edge = (blk + 1) * kBlockKeys > least_lim || page < 0;
    if (edge) {
      POPE_COLD_PATH();
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const int lm = page < 0 ? 0 : lim[n];
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (key0 + 16 * half + i >= lm) s[n][half][i] = -INFINITY;
      }
    }

    // running maximum and sum; P in operand order
    u32x4 pf[NQ];
    float pr[NQ][8];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float mx = fmaxf(fmaxf(fmaxf(s[n][0][0], s[n][0][1]), fmaxf(s[n][0][2], s[n][0][3])),
                       fmaxf(fmaxf(s[n][1][0], s[n][1][1]), fmaxf(s[n][1][2], s[n][1][3])));
      mx = fmaxf(mx, wave_shfl_xor(mx, 16));
      mx = half_swap_max(mx);
      const float mn = fmaxf(m[n], mx);
      const float mu = mn == -INFINITY ? 0.f : mn;
      const float alpha = __builtin_amdgcn_exp2f(m[n] - mu);
      m[n] = mn;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        pr[n][j] = __builtin_amdgcn_exp2f(s[n][j >> 2][j & 3] - mu);
        sum += pr[n][j];
      }
      l[n] = fmaf(l[n], alpha, sum);
#pragma unroll
      for (int v = 0; v < VT; ++v) acc[n][v] *= alpha;
      if constexpr (Q8) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          pr[n][j] = __builtin_amdgcn_ldexpf(pr[n][j], (int)((sv[j >> 2][1] >> (8 * (j & 3))) & 0xff) - 127);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) pf[n][i] = T::pack2(pr[n][2 * i], pr[n][2 * i + 1]);
    }

    // O^T += V^T P^T
    u32x4 va[VT];
#pragma unroll
    for (int v = 0; v < VT; ++v) {
      if constexpr (Q8) va[v] = unpack_e4m3<T>(u32x2{vf[v >> 1][2 * (v & 1)], vf[v >> 1][2 * (v & 1) + 1]}, 1.f);
      else va[v] = vf[v];
    }
    if (edge) {
      POPE_COLD_PATH();
      // slots from len on, and pages outside the cache, hold whatever was there: 0 x NaN must not count
      uint32_t keep = 0, bad = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) keep |= (page >= 0 && key0 + 16 * (j >> 2) + (j & 3) < g.len ? 1u : 0u) << j;
#pragma unroll
      for (int v = 0; v < VT; ++v) {
        va[v] = keep16(va[v], keep);
#pragma unroll
        for (int j = 0; j < 8; ++j) bad |= nonfinite16<T>(va[v][j >> 1] >> (16 * (j & 1))) ? 1u << j : 0u;
      }
      if (__any(bad != 0)) {
        // a value row that some rows do not see is not finite: added outside the product, to the rows that see it
        POPE_COLD_PATH();
        for (int key = 0; key < kBlockKeys; ++key) {
          const int j = 4 * (key >> 4) + (key & 3), from = 16 * ((key & 15) >> 2);
          float pk[NQ];
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            float x = 0.f;
#pragma unroll
            for (int jj = 0; jj < 8; ++jj) x = jj == j ? pr[n][jj] : x;
            pk[n] = __shfl(x, from + col, 64);
          }
#pragma unroll
          for (int v = 0; v < VT; ++v) {
            uint32_t w = 0;
#pragma unroll
            for (int jj = 0; jj < 8; ++jj) w = jj == j ? (va[v][jj >> 1] >> (16 * (jj & 1))) & 0xffffu : w;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t b = (uint32_t)__shfl((int)w, from + quad * 4 + i, 64);
#pragma unroll
              for (int n = 0; n < NQ; ++n)
                if (nonfinite16<T>(b) && blk * kBlockKeys + key < lim[n]) acc[n][v][i] = fmaf(pk[n], T::to_float((uint16_t)b), acc[n][v][i]);
            }
          }
        }
#pragma unroll
        for (int v = 0; v < VT; ++v) {
          uint32_t fin = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) fin |= (nonfinite16<T>(va[v][j >> 1] >> (16 * (j & 1))) ? 0u : 1u) << j;
          va[v] = keep16(va[v], fin);
        }
      }
    }
#pragma unroll
    for (int v = 0; v < VT; ++v)
#pragma unroll
      for (int n = 0; n < NQ; ++n)
        acc[n][v] = T::mfma16(as_vec8<typename T::vec8>(va[v]), as_vec8<typename T::vec8>(pf[n]), acc[n][v]);
    load_v(next_page, next);
    page = next_page;
  }
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    l[n] += wave_shfl_xor(l[n], 16);
    l[n] += wave_shfl_xor(l[n], 32);
  }

  // ---- the waves that share rows join, in a tree over LDS ----------------------------------------------------
  if constexpr (WK > 1) {
    constexpr int kPart = NQ * (VT + 1) * 64;   // f32x4 per wave
    f32x4* join = reinterpret_cast<f32x4*>(smem) + group * (WK / 2) * kPart;
#pragma unroll
    for (int w = WK / 2; w >= 1; w >>= 1) {
      __syncthreads();
      if (wk >= w && wk < 2 * w) {
        f32x4* dst = join + (wk - w) * kPart + lane;
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
#pragma unroll
          for (int v = 0; v < VT; ++v) dst[(n * (VT + 1) + v) * 64] = acc[n][v];
          dst[(n * (VT + 1) + VT) * 64] = f32x4{m[n], l[n], 0.f, 0.f};
        }
      }
      __syncthreads();
      if (wk < w) {
        const f32x4* src = join + wk * kPart + lane;
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          const f32x4 ml = src[(n * (VT + 1) + VT) * 64];
          const float mn = fmaxf(m[n], ml[0]), mu = mn == -INFINITY ? 0.f : mn;
          const float a = __builtin_amdgcn_exp2f(m[n] - mu), b = __builtin_amdgcn_exp2f(ml[0] - mu);
          m[n] = mn;
          l[n] = l[n] * a + ml[1] * b;
#pragma unroll
          for (int v = 0; v < VT; ++v) acc[n][v] = acc[n][v] * a + src[(n * (VT + 1) + v) * 64] * b;
        }
      }
    }
    if (wk) return;
  }

  // ---- output, or this split's part ---------------------------------------------------------------------------
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    if (!live[n]) continue;
    if (part) {
      const int64_t row = (((int64_t)tile * c.Hk + hk) * p.splits + split) * kRows + group * 16 * NQ + n * 16 + col;
      float* dst = p.part_o + row * (VT * 16) + quad * 4;
#pragma unroll
      for (int v = 0; v < VT; ++v) *reinterpret_cast<f32x4*>(dst + v * 16) = acc[n][v];
      if (quad == 0) *reinterpret_cast<float2*>(p.part_ml + row * 2) = make_float2(m[n], l[n]);
      continue;
    }
    const float inv = l[n] == 0.f ? 0.f : 1.f / l[n];
    uint16_t* dst = p.o + (int64_t)g.batch * p.o_s[0] + (int64_t)row_h[n] * p.o_s[1] + (int64_t)(g.row0 + row_i[n]) * p.o_s[2];
#pragma unroll
    for (int v = 0; v < VT; ++v) {
      const int d = v * 16 + quad * 4;
      const f32x4 x = acc[n][v] * inv;
      if (p.o_vec) {
        if (d < c.D) *reinterpret_cast<u32x2*>(dst + d) = u32x2{T::pack2(x[0], x[1]), T::pack2(x[2], x[3])};
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (d + i < c.D) dst[d + i] = T::bits(x[i]);
      }
    }
    if (p.lse && quad == 0)
      p.lse[((int64_t)g.batch * p.Hq + row_h[n]) * p.N + g.row0 + row_i[n]] =
          l[n] == 0.f ? -INFINITY : (m[n] + __builtin_amdgcn_logf(l[n])) * kLn2;
  }
}

// The splits' parts of a tile's rows joined: a thread has four columns of a row, and keeps a running (m, l, o).
template <typename T, int VT>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnParams p, int rows, int step) {
  const PagedCache& c = p.c;
  const int hk = blockIdx.x % c.Hk, tile = blockIdx.x / c.Hk;
  const PagedTile t = paged_tile(c.seqs, tile, p.G.d, rows, 1);
  const PagedSeg& g = t.seg;
  const int rows_all = g.n * (int)p.G.d, r0 = t.local * rows;
  if (r0 >= rows_all) return;
  const int blocks = paged_tile_blocks(g, t.local, rows, p.G, p.causal != 0);
  const int parts = paged_parts(blocks, p.splits, p.least, step);
  if (parts <= 1) return;   // written by the one that had it
  constexpr int kCols = VT * 4;   // threads per row
  for (int it = blockIdx.y * 256 + threadIdx.x; it < rows * kCols; it += gridDim.y * 256) {
    const int rr = it / kCols, d = it % kCols * 4;
    const int r = r0 + rr;
    if (r >= rows_all || d >= c.D) continue;
    const int64_t first = ((int64_t)tile * c.Hk + hk) * p.splits * (int64_t)rows + rr;
    float m = -INFINITY, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < parts; ++s) {
      const int64_t row = first + (int64_t)s * rows;
      const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + row * 2);
      const f32x4 x = *reinterpret_cast<const f32x4*>(p.part_o + row * (VT * 16) + d);
      const float mn = fmaxf(m, ml.x), mu = mn == -INFINITY ? 0.f : mn;
      const float a = __builtin_amdgcn_exp2f(m - mu), b = __builtin_amdgcn_exp2f(ml.x - mu);
      m = mn;
      l = l * a + ml.y * b;
      o = o * a + x * b;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int i = (int)p.G.of(r), h = (r - i * (int)p.G.d) * c.Hk + hk;
    uint16_t* dst = p.o + (int64_t)g.batch * p.o_s[0] + (int64_t)h * p.o_s[1] + (int64_t)(g.row0 + i) * p.o_s[2] + d;
    if (p.o_vec) {
      *reinterpret_cast<u32x2*>(dst) = u32x2{T::pack2(o[0] * inv, o[1] * inv), T::pack2(o[2] * inv, o[3] * inv)};
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (d + k < c.D) dst[k] = T::bits(o[k] * inv);
    }
    if (p.lse && d == 0)
      p.lse[((int64_t)g.batch * p.Hq + h) * p.N + g.row0 + i] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
  }
}

template <typename T, bool Q8, int KS, int VT, int NQ, int WK>
hipError_t run_paged_attn(const PagedAttnParams& p, hipStream_t s) {
  constexpr int rows = 16 * NQ * (4 / WK);
  const int64_t wgs = p.tiles * p.c.Hk * p.splits;
  hipError_t e = launch_named("paged_attn", paged_attn_kernel<T, Q8, KS, VT, NQ, WK>, dim3((unsigned)wgs), dim3(256), s, p);
  if (e != hipSuccess || p.splits == 1) return e;
  const int y = (rows * VT * 4 + 255) / 256;
  return launch_named("paged_join", paged_join_kernel<T, VT>, dim3((unsigned)(p.tiles * p.c.Hk), y), dim3(256), s, p, rows, WK);
}

template <typename T, bool Q8, int KS, int VT>
hipError_t run_paged_rows(const PagedAttnParams& p, hipStream_t s) {
  constexpr int rows = PagedRows<Q8, KS, VT>::kRows;
  const int64_t wgs = p.tiles * p.c.Hk * p.splits;
  const hipError_t e = launch_named("paged_rows", paged_rows_kernel<T, Q8, KS, VT>, dim3((unsigned)wgs), dim3(256), s, p);
  if (e != hipSuccess || p.splits == 1) return e;
  const int y = (rows * VT * 4 + 255) / 256;
  return launch_named("paged_join", paged_join_kernel<T, VT>, dim3((unsigned)(p.tiles * p.c.Hk), y), dim3(256), s, p, rows, 1);
}

template <typename T, bool Q8, int KS, int VT>
hipError_t run_paged_plan(const PagedAttnParams& p, PagedPlan plan, hipStream_t s) {
  if (plan.wk == 4 && plan.nq == 1) return run_paged_attn<T, Q8, KS, VT, 1, 4>(p, s);
  if constexpr (VT > 8) return run_paged_attn<T, Q8, KS, VT, 1, 1>(p, s);   // paged_plan
  else return plan.wk == 4 ? run_paged_attn<T, Q8, KS, VT, 2, 4>(p, s) : run_paged_rows<T, Q8, KS, VT>(p, s);
}

// The instance of (steps, tiles): paged_k_steps and paged_v_tiles give no other.
template <typename T, bool Q8>
hipError_t run_paged_shape(const PagedAttnParams& p, PagedPlan plan, hipStream_t s) {
#define POPE_PAGED(KS, VT) \
  if (p.c.steps == KS && p.c.tiles == VT) return run_paged_plan<T, Q8, KS, VT>(p, plan, s);
  POPE_PAGED(1, 2) POPE_PAGED(2, 2)
  POPE_PAGED(2, 4) POPE_PAGED(3, 4) POPE_PAGED(4, 4)
  POPE_PAGED(3, 6) POPE_PAGED(5, 6) POPE_PAGED(6, 6)
  POPE_PAGED(4, 8) POPE_PAGED(6, 8) POPE_PAGED(8, 8)
  POPE_PAGED(8, 16) POPE_PAGED(12, 16) POPE_PAGED(16, 16)
#undef POPE_PAGED
  return hipErrorInvalidValue;
}

}  // namespace pope
