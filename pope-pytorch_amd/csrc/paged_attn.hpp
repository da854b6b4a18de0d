// Attention of new tokens over the paged cache (gfx950): this kernel for up to 16 rows of a key head (single tokens, a few
// proposed ones, grouped heads), paged_rows.hpp for more.
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
// passes through LDS: a wave streams 1 KB loads into registers, the next block's while it works on this one's.  Row sums
// and maxima of a row lie in the four lanes l % 16.
//
// Bound by HBM.  The four waves of a workgroup take every fourth block of 32 keys and join through LDS; where the tiles
// leave the chip idle, workgroups take parts of the key axis, and a second launch joins those that had several.
// Measured: 8 sequences of 4,096 .. 32,768 tokens, 16 heads, D 64, R 64, 16 bits, 906 MB: 165 us with the join, 5.5 TB/s
// (a copy: 4.7, half of it writes); 32 of 1,000 .. 16,384, 8 key heads of 4 query heads, D 128, R 64, 8 bits, 717 MB: 155 us,
// 4.6 TB/s.  One sequence of 4,000 tokens, 18 MB: 13 us, two launches and a wave's chain of a few blocks.
//
// Precision: S, the maxima, sums and O in fp32.  Q_hat is the sum of two 16-bit parts (twice the S products: rounded once, its
// error would appear in every score, about 0.8 of an output's own rounding at N(0, 1) inputs), and so is P here, where
// products are free: what is left is the output's rounding.
#pragma once
#include "paged_rows.hpp"

namespace pope {

template <int KS, int VT>
struct PagedFew {
  static constexpr int kRows = 16, kWaves = 4;
  static constexpr int QST = KS * 32 + 8;                          // row stride of Q_hat in LDS: an odd number of 16-byte units
  static constexpr int kQ = 2 * kRows * QST * 2, kJoin = kWaves / 2 * (VT + 1) * 64 * 16;
  static constexpr int kBytes = kQ > kJoin ? kQ : kJoin;
};

template <typename T, bool Q8, int KS, int VT>
__global__ __launch_bounds__(256, VT <= 8 ? 2 : 1) void paged_few_kernel(PagedAttnParams p) {
  using C = PagedFew<KS, VT>;
  typedef typename T::vec8 vec8;
  typedef std::conditional_t<Q8, BF16, T> V;   // the second product's: P x 2^e leaves fp16's range where values are far from 1
  constexpr int kRows = C::kRows, WK = C::kWaves, QST = C::QST;
  __shared__ __attribute__((aligned(16))) char smem[C::kBytes];
  const PagedCache& c = p.c;
  const int lane = threadIdx.x & 63, wave = wave_id(), col = lane & 15, quad = lane >> 4;

  const PagedJob job = paged_job(p);
  const int hk = job.hk;
  const PagedTile t = paged_tile(c.seqs, job.tile, p.G.d, kRows, 1);
  const PagedSeg& g = t.seg;
  const int rows_all = g.n * (int)p.G.d, r0 = t.local * kRows;
  if (r0 >= rows_all) return;
  const bool causal = p.causal != 0;
  const int blocks = paged_tile_blocks(g, t.local, kRows, p.G, causal);
  const int least = paged_few_least(blocks, p.tiles * c.Hk);
  const PagedRange range = paged_range(blocks, p.splits, least, WK, job.split);
  const int parts = paged_parts(blocks, p.splits, least, WK);
  if (job.split > 0 && range.begin >= range.end) return;
  if (p.splits > 1 && job.split == 0 && threadIdx.x == 0) p.parts[(int64_t)job.tile * c.Hk + hk] = parts;
  const bool part = parts > 1;

  // ---- the first block's loads ---------------------------------------------------------------------------------
  constexpr int kKL = Q8 ? KS : 2 * KS, kVL = Q8 ? VT / 2 : VT, kE = Q8 ? 1 : 2;   // 16-byte loads per lane and block; bytes
  // page numbers of 64 pages at a time, one per lane; -1: outside the cache
  int page_base = 0, pids = 0;
  auto page_of = [&](int blk) {
    const int pg = blk >> c.blk_shift;
    if (pg - page_base >= 64) {
      page_base = pg;
      const int cols = c.seqs.capacity >> (c.blk_shift + 5);
      const int id = c.table[(int64_t)g.b * c.table_sb + min(pg + lane, cols - 1)];
      pids = (unsigned)id < (unsigned)c.pages ? id : -1;
    }
    return __builtin_amdgcn_readlane(pids, pg - page_base);
  };
  u32x4 kf[kKL], vf[kVL];
  u32x2 sk[2];   // exponent bytes (8-bit caches): [K0..3][V0..3] of the lane's keys of either half
  // operands of a block; a page outside the cache reads page 0 and is masked
  auto load_k = [&](int page, int blk) {
    const int pg = max(page, 0);
    const char* base = static_cast<const char*>(c.k) + paged_block_off(c, pg, hk, blk, c.k_head, KS * 1024) * kE + lane * 16;
#pragma unroll
    for (int i = 0; i < kKL; ++i) kf[i] = *reinterpret_cast<const u32x4*>(base + i * 1024);
    if constexpr (Q8) {
      const uint8_t* s = c.scales + paged_scale_base(c, pg, hk, blk) + quad * 8;
      sk[0] = *reinterpret_cast<const u32x2*>(s);
      sk[1] = *reinterpret_cast<const u32x2*>(s + 32);
    }
  };
  auto load_v = [&](int page, int blk) {
    const char* base = static_cast<const char*>(c.v) + paged_block_off(c, max(page, 0), hk, blk, c.v_head, VT * 512) * kE + lane * 16;
#pragma unroll
    for (int i = 0; i < kVL; ++i) vf[i] = *reinterpret_cast<const u32x4*>(base + i * 1024);
  };

  // ---- the lane's row ------------------------------------------------------------------------------------------
  const PagedRowMap map(r0, p.G);
  const int count = min(rows_all - r0, kRows);
  const bool live = col < count;
  const int row_i = live ? map.token(col) : 0, row_h = live ? map.group(col) * c.Hk + hk : hk;
  const int lim = live ? paged_limit(g.first + row_i, g.len, causal) : 0;
  const int least_lim = paged_limit(g.first + (int)map.i0, g.len, causal);   // the first row sees the fewest keys

  int blk = range.begin + wave, page = -1;
  PagedQueryIn in[(VT + 7) / 8];
#pragma unroll
  for (int k = 0; k < (VT + 7) / 8; ++k) in[k] = paged_query_load<T>(p, g, map, (threadIdx.x + 256 * k) % kRows, count, hk, (threadIdx.x + 256 * k) / kRows * 8);
  if (blk < range.end) {
    page_base = -(1 << 20);
    page = page_of(blk);
    load_k(page, blk);
    load_v(page, blk);
  }

  // ---- Q_hat, through LDS --------------------------------------------------------------------------------------
  vec8 qh[KS], ql[KS];
  {
    uint16_t* hi = reinterpret_cast<uint16_t*>(smem);
    uint16_t* lo = hi + kRows * QST;
#pragma unroll
    for (int k = 0; k < (VT + 7) / 8; ++k) paged_query_make<T>(p, in[k], true, (threadIdx.x + 256 * k) % kRows, (threadIdx.x + 256 * k) / kRows * 8, QST, hi, lo);
    paged_query_tail<kRows>(p, threadIdx.x, 256, KS * 32, QST, hi, lo);
    __syncthreads();
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qh[ks] = as_vec8<vec8>(*reinterpret_cast<const u32x4*>(hi + col * QST + ks * 32 + quad * 8));
      ql[ks] = as_vec8<vec8>(*reinterpret_cast<const u32x4*>(lo + col * QST + ks * 32 + quad * 8));
    }
  }

  // ---- the loop over the wave's blocks -----------------------------------------------------------------------
  f32x4 acc[VT];
#pragma unroll
  for (int v = 0; v < VT; ++v) acc[v] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  auto exponent = [](uint32_t w, int i) { return (int)((w >> (8 * i)) & 0xffu) - 127; };
  // a block's running maximum and sum; P in operand order, in two parts; O^T += V^T P^T
  float pr[8];
  auto attend = [&](const f32x4* s, const uint32_t* sv) __attribute__((always_inline)) {
    float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    mx = fmaxf(mx, wave_shfl_xor(mx, 16));
    mx = half_swap_max(mx);
    const float mn = fmaxf(m, mx), mu = mn == -INFINITY ? 0.f : mn, alpha = __builtin_amdgcn_exp2f(m - mu);
    m = mn;
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      pr[j] = __builtin_amdgcn_exp2f(s[j >> 2][j & 3] - mu);
      sum += pr[j];
      if (Q8) pr[j] = __builtin_amdgcn_ldexpf(pr[j], exponent(sv[j >> 2], j & 3));
    }
    l = fmaf(l, alpha, sum);
    u32x4 ph, pl;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ph[i] = V::pack2(pr[2 * i], pr[2 * i + 1]);
      pl[i] = V::pack2(pr[2 * i] - V::to_float((uint16_t)ph[i]), pr[2 * i + 1] - V::to_float((uint16_t)(ph[i] >> 16)));
    }
#pragma unroll
    for (int v = 0; v < VT; ++v) {
      typename V::vec8 a;
      if constexpr (Q8) a = as_vec8<typename V::vec8>(unpack_e4m3<V>(u32x2{vf[v >> 1][2 * (v & 1)], vf[v >> 1][2 * (v & 1) + 1]}, 1.f));
      else a = as_vec8<typename V::vec8>(vf[v]);
      acc[v] *= alpha;
      acc[v] = V::mfma16(a, as_vec8<typename V::vec8>(ph), acc[v]);
      acc[v] = V::mfma16(a, as_vec8<typename V::vec8>(pl), acc[v]);
    }
  };
  // the values that are not finite of the keys in `odd`, where they are seen
  auto add_seen = [&](int page, int blk, uint32_t odd) __attribute__((always_inline)) {
    const int64_t at = paged_block_off(c, max(page, 0), hk, blk, c.v_head, VT * 512);
#pragma unroll 1
    for (int key = 0; key < kBlockKeys; ++key) {
      if (!__any((odd >> key) & 1)) continue;
      const int j = 4 * (key >> 4) + (key & 3);
      float pk = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) pk = k == j ? pr[k] : pk;
      pk = __shfl(pk, col + 16 * ((key & 15) >> 2), 64);
      const bool seen = blk * kBlockKeys + key < lim;
#pragma unroll
      for (int v = 0; v < VT; ++v) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t off = at + paged_v_off(Q8, key, v * 16 + quad * 4 + i);
          const uint32_t w = Q8 ? ((static_cast<const uint8_t*>(c.v)[off] & 0x7f) == 0x7f ? 0x7fffu : 0u) : static_cast<const uint16_t*>(c.v)[off];
          if (nonfinite16<T>(w) && seen) acc[v][i] = fmaf(pk, T::to_float((uint16_t)w), acc[v][i]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  // The wave's blocks once more, for rows that infinite keys or values made NaN (paged_dev.hpp).
  auto second_pass = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int v = 0; v < VT; ++v) acc[v] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.f;
#pragma unroll 1
    for (int blk = range.begin + wave; blk < range.end; blk += WK) {
      const int page = paged_page(c, g.b, blk);
      if (page < 0) continue;
      const char* keys = static_cast<const char*>(c.k) + paged_block_off(c, page, hk, blk, c.k_head, KS * 1024) * kE + lane * 16;
      f32x4 s[2], lo[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) s[half] = lo[half] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          u32x4 fin, rest;
          split_finite<T>(*reinterpret_cast<const u32x4*>(keys + (2 * ks + half) * 1024), &fin, &rest);
          s[half] = T::mfma16(as_vec8<vec8>(fin), qh[ks], s[half]);
          lo[half] = T::mfma16(as_vec8<vec8>(fin), ql[ks], lo[half]);
          if (__any((rest[0] | rest[1] | rest[2] | rest[3]) != 0)) lo[half] = T::mfma16(as_vec8<vec8>(rest), sign_operand<T>(qh[ks]), lo[half]);
        }
      const int key0 = blk * kBlockKeys + quad * 4;
      const uint32_t sv[2] = {0, 0};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        s[half] += lo[half];
        if (T::kCode == 1) s[half] *= p.late;
#pragma unroll
        for (int i = 0; i < 4; ++i) s[half][i] = key0 + 16 * half + i < lim ? s[half][i] : -INFINITY;
      }
      uint32_t odd = 0;
      load_v(page, blk);
#pragma unroll
      for (int v = 0; v < kVL; ++v) clean_values<T, Q8>(vf[v], g.len - key0, 4 * quad, odd);
      attend(s, sv);
      add_seen(page, blk, odd);
    }
  };
  for (; blk < range.end; blk += WK) {
    const int next = blk + WK < range.end ? blk + WK : blk;   // the last one is loaded again, unused
    const int next_page = page_of(next);

    // S^T of the block's two key halves: the parts of Q_hat in chains of their own
    f32x4 s[2], lo[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) s[half] = lo[half] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        vec8 a;
        if constexpr (Q8) a = as_vec8<vec8>(unpack_e4m3<T>(u32x2{kf[ks][2 * half], kf[ks][2 * half + 1]}, 1.f));
        else a = as_vec8<vec8>(kf[2 * ks + half]);
        s[half] = T::mfma16(a, qh[ks], s[half]);
        lo[half] = T::mfma16(a, ql[ks], lo[half]);
      }
    uint32_t sv[2] = {0, 0};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      s[half] += lo[half];
      if constexpr (Q8) {
        sv[half] = sk[half][1];
#pragma unroll
        for (int i = 0; i < 4; ++i) s[half][i] = __builtin_amdgcn_ldexpf(s[half][i], exponent(sk[half][0], i));
      }
      if (T::kCode == 1) s[half] *= p.late;
    }
    load_k(next_page, next);

    const int key0 = blk * kBlockKeys + quad * 4;   // the lane's keys: key0 + 16 half + i
    const bool edge = (blk + 1) * kBlockKeys > least_lim || page < 0;
    uint32_t odd = 0;   // keys of the block whose values are not finite, where some row may not see them
    if (edge) {
      POPE_COLD_PATH();
      const int lm = page < 0 ? 0 : lim, have = page < 0 ? 0 : g.len - key0;
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[half][i] = key0 + 16 * half + i < lm ? s[half][i] : -INFINITY;
      // Slots from len on, and pages outside the cache, hold whatever was there: 0 x NaN must not count.  They become
      // zeros; so do values that are not finite, whose keys are noted and which are added below where they are seen.
#pragma unroll
      for (int v = 0; v < kVL; ++v) clean_values<T, Q8>(vf[v], have, 4 * quad, odd);
    }
    attend(s, sv);
    load_v(next_page, next);
    if (edge && __any(odd != 0)) {
      POPE_COLD_PATH();
      add_seen(page, blk, odd);
    }
    page = next_page;
  }
  if constexpr (!Q8) {
    float x = l;
#pragma unroll
    for (int v = 0; v < VT; ++v) x += (acc[v][0] + acc[v][1]) + (acc[v][2] + acc[v][3]);
    if (__builtin_expect(__any(x != x), 0)) {
      POPE_COLD_PATH();
      bool fin = true;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) fin = fin && all_finite<T>(qh[ks]);
      const uint64_t nan = __ballot(x != x && live), off = __ballot(!fin);   // of a row: in any of its four lanes
      const auto of_row = [&](uint64_t w) { return (w | w >> 16 | w >> 32 | w >> 48) & 0xffffu; };
      if (of_row(nan) & ~of_row(off)) second_pass();
    }
  }
  l += wave_shfl_xor(l, 16);
  l += wave_shfl_xor(l, 32);

  // ---- the waves join, in a tree over LDS ----------------------------------------------------------------------
  constexpr int kPart = (VT + 1) * 64;   // f32x4 per wave
  f32x4* join = reinterpret_cast<f32x4*>(smem);
#pragma unroll
  for (int w = WK / 2; w >= 1; w >>= 1) {
    __syncthreads();
    if (wave >= w && wave < 2 * w) {
      f32x4* dst = join + (wave - w) * kPart + lane;
#pragma unroll
      for (int v = 0; v < VT; ++v) dst[v * 64] = acc[v];
      dst[VT * 64] = f32x4{m, l, 0.f, 0.f};
    }
    __syncthreads();
    if (wave < w) {
      const f32x4* src = join + wave * kPart + lane;
      const f32x4 ml = src[VT * 64];
      const float mn = fmaxf(m, ml[0]), mu = mn == -INFINITY ? 0.f : mn;
      const float a = __builtin_amdgcn_exp2f(m - mu), b = __builtin_amdgcn_exp2f(ml[0] - mu);
      m = mn;
      l = l * a + ml[1] * b;
#pragma unroll
      for (int v = 0; v < VT; ++v) acc[v] = acc[v] * a + src[v * 64] * b;
    }
  }
  if (wave || !live) return;

  // ---- output, or this split's part ----------------------------------------------------------------------------
  const int64_t row = (((int64_t)job.tile * c.Hk + hk) * kRows + col) * p.splits + job.split;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* dst = p.o + (int64_t)g.batch * p.o_s[0] + (int64_t)row_h * p.o_s[1] + (int64_t)(g.row0 + row_i) * p.o_s[2];
#pragma unroll
  for (int v = 0; v < VT; ++v) {
    const int d = v * 16 + quad * 4;
    const f32x4 x = part ? acc[v] : averages<T>(acc[v] * inv);
    if (part) {
      *reinterpret_cast<f32x4*>(p.part_o + row * (VT * 16) + d) = x;
    } else if (p.o_vec) {
      if (d < c.D) *reinterpret_cast<u32x2*>(dst + d) = u32x2{T::pack2(x[0], x[1]), T::pack2(x[2], x[3])};
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (d + i < c.D) dst[d + i] = T::bits(x[i]);
    }
  }
  if (quad == 0) {
    if (part) *reinterpret_cast<float2*>(p.part_ml + row * 2) = make_float2(m, l);
    else if (p.lse)
      p.lse[((int64_t)g.batch * p.Hq + row_h) * p.N + g.row0 + row_i] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
  }
}

// The parts of a tile's rows joined, RPW rows per workgroup.  A thread has four columns of a row and every kGroups-th of its
// parts, of which it keeps a running (m, l, o); the groups join through LDS.  A row's parts lie side by side.
template <typename T, int VT, int RPW>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnParams p, int rows) {
  constexpr int kQuads = VT * 4, kGroups = 256 / (RPW * kQuads);
  __shared__ f32x4 o_s[256];
  __shared__ float2 ml_s[256];
  const PagedCache& c = p.c;
  const int hk = blockIdx.x % c.Hk, tile = blockIdx.x / c.Hk, tid = threadIdx.x;
  const PagedTile t = paged_tile(c.seqs, tile, p.G.d, rows, 1);
  const PagedSeg& g = t.seg;
  const int count = min(g.n * (int)p.G.d - t.local * rows, rows);
  if ((int)blockIdx.y * RPW >= count) return;
  // bounded: lengths that another stream changes between the launches must not lead out of the workspace
  const int parts = min(p.parts[blockIdx.x], p.splits);
  if (parts <= 1) return;   // written by the one that had it
  const int d = tid % kQuads * 4, group = tid / (kQuads * RPW);
  for (int r0 = blockIdx.y * RPW; r0 < count; r0 += gridDim.y * RPW) {
    const int rr = r0 + tid / kQuads % RPW;
    const bool on = group < kGroups && rr < count && d < c.D;
    float m = -INFINITY, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    // a part whose scores are all NaN has m = -inf, as one without a visible key, but l = NaN, and its row becomes NaN
    auto fold = [&](float2 ml, f32x4 x) {
      const float mn = fmaxf(m, ml.x), mu = mn == -INFINITY ? 0.f : mn;
      const float a = __builtin_amdgcn_exp2f(m - mu), b = __builtin_amdgcn_exp2f(ml.x - mu);
      m = mn;
      l = l * a + ml.y * b;
      o = o * a + x * b;
    };
    if (on) {
      const int64_t first = (((int64_t)tile * c.Hk + hk) * rows + rr) * p.splits;
#pragma unroll 4
      for (int s = group; s < parts; s += kGroups)
        fold(*reinterpret_cast<const float2*>(p.part_ml + (first + s) * 2), *reinterpret_cast<const f32x4*>(p.part_o + (first + s) * (VT * 16) + d));
    }
    if constexpr (kGroups > 1) {
      __syncthreads();   // the rows before have been read
      o_s[tid] = o;
      ml_s[tid] = make_float2(m, l);
      __syncthreads();
      if (on && group == 0) {
#pragma unroll
        for (int k = 1; k < kGroups; ++k) fold(ml_s[tid + k * kQuads * RPW], o_s[tid + k * kQuads * RPW]);
      }
    }
    if (!on || group) continue;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int r = t.local * rows + rr, i = (int)p.G.of(r), h = (r - i * (int)p.G.d) * c.Hk + hk;
    uint16_t* dst = p.o + (int64_t)g.batch * p.o_s[0] + (int64_t)h * p.o_s[1] + (int64_t)(g.row0 + i) * p.o_s[2] + d;
    const f32x4 x = averages<T>(o * inv);
    if (p.o_vec) {
      *reinterpret_cast<u32x2*>(dst) = u32x2{T::pack2(x[0], x[1]), T::pack2(x[2], x[3])};
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (d + k < c.D) dst[k] = T::bits(x[k]);
    }
    if (p.lse && d == 0)
      p.lse[((int64_t)g.batch * p.Hq + h) * p.N + g.row0 + i] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
  }
}

template <typename T, bool Q8, int KS, int VT>
hipError_t run_paged_plan(const PagedAttnParams& p, bool few, hipStream_t s) {
  constexpr int least_rows = PagedFew<KS, VT>::kRows, most_rows = PagedRows<Q8, KS, VT>::kRows;
  static_assert(least_rows == kPagedFewRows && most_rows == kPagedManyRows, "tiles as the host counts them");
  const dim3 grid((unsigned)(p.tiles * p.c.Hk * p.splits));
  const hipError_t e = few ? launch_named("paged_few", paged_few_kernel<T, Q8, KS, VT>, grid, dim3(256), s, p)
                           : launch_named("paged_rows", paged_rows_kernel<T, Q8, KS, VT>, grid, dim3(256), s, p);
  if (e != hipSuccess || p.splits == 1) return e;
  // Rows at a time, and workgroups per tile: about 2,048 in all, since finding the tile costs one as much as its rows do
  // (4,096-token prompts, 2 x 8 heads: 16,384 workgroups of 4 rows took 20 us).
  constexpr int few_rpw = VT <= 8 ? 4 : 1, many_rpw = VT < 8 ? 4 : VT == 8 ? 8 : 4;
  const int64_t heads = p.tiles * p.c.Hk, each = 2048 / heads;
  const auto y = [&](int most) { return (unsigned)(each < 1 ? 1 : each < most ? each : most); };
  if (few) return launch_named("paged_join", paged_join_kernel<T, VT, few_rpw>, dim3((unsigned)heads, y(least_rows / few_rpw)), dim3(256), s, p, least_rows);
  return launch_named("paged_join", paged_join_kernel<T, VT, many_rpw>, dim3((unsigned)heads, y(most_rows / many_rpw)), dim3(256), s, p, most_rows);
}

// The instance of (steps, tiles): paged_k_steps and paged_v_tiles give no other.
template <typename T, bool Q8>
hipError_t run_paged_shape(const PagedAttnParams& p, bool few, hipStream_t s) {
#define POPE_PAGED(KS, VT) \
  if (p.c.steps == KS && p.c.tiles == VT) return run_paged_plan<T, Q8, KS, VT>(p, few, s);
  POPE_PAGED(1, 2) POPE_PAGED(2, 2)
  POPE_PAGED(2, 4) POPE_PAGED(3, 4) POPE_PAGED(4, 4)
  POPE_PAGED(3, 6) POPE_PAGED(5, 6) POPE_PAGED(6, 6)
  POPE_PAGED(4, 8) POPE_PAGED(6, 8) POPE_PAGED(8, 8)
  POPE_PAGED(8, 16) POPE_PAGED(12, 16) POPE_PAGED(16, 16)
#undef POPE_PAGED
  return hipErrorInvalidValue;
}

}  // namespace pope
