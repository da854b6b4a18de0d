// States of the linear attention between segments, and the phases' gradients (gfx950).
//
//   states   what the rows of a segment add to the state behind it, sum_j g^(len-1-j) k_hat_j v_j^T, or, in reverse, to the
//            gradient of the state before it, sum_i g^(i+1) scale q_hat_i dO_i^T
//   scan     S <- g^len S + sum, segment by segment; what a segment starts from goes where its sum was
//   phase    sums of the phases' gradients over segments (bias) and heads (freqs), in a fixed order
//
// The sums come out as fp32 states, so each expanded row goes in as the sum of two bf16 parts, weighted in fp32 before it is
// split: 2^-17 of each product.
#include "linear_dev.hpp"

namespace pope {

namespace {

template <typename T, typename K>
__global__ __launch_bounds__(K::kThreads, 1) void linear_state_kernel(LinStateParams p) {
  constexpr int NT = K::NT, CT = K::CT, PL = K::PL, C = K::C, KS = K::KS, ST = K::P / 32;
  __shared__ __attribute__((aligned(16))) uint16_t lds[2 * C * K::YS + PL * C * K::ZS];
  __shared__ float turns[256];
  const LinCall& c = p.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), q4 = lane >> 4, l16 = lane & 15;
  const int wg = blockIdx.x, tile = wg % p.tiles, rest = wg / p.tiles, hk = rest % c.Hk, at = rest / c.Hk;
  const LinSeg seg = lin_segment(c.seqs, at);
  if (seg.seq < 0) return;
  const LinTile Y{lds, K::YS, C * K::YS}, Z{lds + 2 * C * K::YS, K::ZS, C * K::ZS};
  for (int i = tid; i < (int)sizeof(lds) / 16; i += K::kThreads) reinterpret_cast<u32x4*>(lds)[i] = u32x4{0, 0, 0, 0};
  const bool rev = p.reverse != 0;
  if (!rev)
    for (int d = tid; d < c.R; d += K::kThreads) turns[d] = lin_turns(c.bias[hk * c.bias_sh + d]);
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
  const int tz = (C * ((min(NT, c.Dv) + 31) / 32 * 4) + K::kThreads - 1) / K::kThreads;
  typedef LinItem<C, K::kThreads> Item;
  for (int t0 = 0; t0 < seg.len; t0 += C)
    for (int g = 0; g < G; ++g) {
      const int h = rev ? g * c.Hk + hk : hk;
      __syncthreads();   // nothing reads the tiles any more
#pragma unroll 2
      for (int u = 0; u < ty; ++u) {
        const Item i(u);
        if (i.d0 >= c.D) continue;
        const int row = seg.row0 + t0 + i.row;
        u32x4 x = {0, 0, 0, 0};
        f32x4 f[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        const bool live = t0 + i.row < seg.len && (rev || !c.mask || c.mask[(int64_t)seg.batch * c.mask_sb + row]);
        if (live) {
          x = lin_load8(yr.p + (int64_t)seg.batch * yr.s[0] + (int64_t)h * yr.s[1] + (int64_t)row * yr.s[2], i.d0, c.D, yr.vec);
          if (c.R) lin_angles8(lin_angle_row(c, seg.batch, row), i.d0, c.R, c.f_vec, f);
        }
        const int n = rev ? t0 + i.row + 1 : seg.len - 1 - t0 - i.row;
        lin_put_polar<T, 2, false>(Y, i.row, i.d0, x, f, live, live ? lin_power(lg, n) * (rev ? c.scale : 1.f) : 0.f, bias, c.D, c.R, 0, K::P);
      }
#pragma unroll 2
      for (int u = 0; u < tz; ++u) {
        const Item i(u);
        if (i.d0 >= NT || n0 + i.d0 >= c.Dv) continue;
        const int row = seg.row0 + t0 + i.row;
        u32x4 x = {0, 0, 0, 0};
        if (t0 + i.row < seg.len && (rev || !c.mask || c.mask[(int64_t)seg.batch * c.mask_sb + row]))
          x = lin_load8(zr.p + (int64_t)seg.batch * zr.s[0] + (int64_t)h * zr.s[1] + (int64_t)row * zr.s[2], n0 + i.d0, c.Dv, zr.vec);
        lin_put_plain<T, PL, false>(Z, i.row, i.d0, x);
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
  if (!busy) return;
  float* to = p.states + ((int64_t)at * c.Hk + hk) * c.E * c.Dv;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int col = n0 + col0 + 16 * ct + l16;
#pragma unroll
    for (int s = 0; s < 2 * ST; ++s)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * s + 4 * q4 + r;
        if (row < c.E && col < c.Dv) to[(int64_t)row * c.Dv + col] = W[ct][s][r];
      }
  }
}

template <typename T>
struct StateLaunch {
  template <typename K>
  struct Of {
    static hipError_t go(LinStateParams p, hipStream_t s) {
      p.tiles = (p.c.Dv + K::NT - 1) / K::NT;
      const int64_t n = (int64_t)p.c.seqs.T * p.c.Hk * p.tiles;
      if (n >= ((int64_t)1 << 22)) return hipErrorInvalidValue;
      return launch_named("linear_states", linear_state_kernel<T, K>, dim3((unsigned)n), dim3(K::kThreads), s, p);
    }
  };
};

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
  if (q == 0 && d < c.R) p.dbias[(int64_t)h0 * c.R + d] = (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
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

hipError_t launch_linear_states(const LinStateParams& p, int dtype, hipStream_t s) {
  return dtype == BF16::kCode ? lin_dispatch<BF16, StateLaunch<BF16>::Of>(p.c.E, p.c.Dv, p, s) : lin_dispatch<F16, StateLaunch<F16>::Of>(p.c.E, p.c.Dv, p, s);
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
