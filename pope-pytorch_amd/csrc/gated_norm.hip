// Norm of head rows with a gate (gfx950): y = x r w silu(gate), r = 1 / sqrt(mean x^2 + eps), and its gradients
//   t = dy w silu(gate),  dx = r (t - x r^2 mean(t x)),  dgate = dy x r w silu'(gate),  dw = sum over rows of dy x r silu(gate)
//
// Bound by HBM (three rows of 16-bit values forward, five backward) or the launch.  A row is 8 columns for each of 8 to 64 lanes;
// all arithmetic is fp32, rounded once.
// 48,000 rows of 128 with fp32 x: 14 us (3.5 TB/s) and 21 back (3.9); 96,000 rows of 100 in fp16, in units of four: 16 us, 3.6 TB/s
// (element by element 34); 65,536 rows of 64: 11 and 17, which is latency: four turns of a workgroup, each waiting for its rows.
#include <algorithm>

#include "linear_dev.hpp"

namespace pope {

namespace {

constexpr int kThreads = 256;
constexpr int kNormGrid = 2048, kNormRows = 4;   // workgroups that fill the chip; the least turns of one

// Eight elements from column d0 on; r.vec: whole aligned units of 8, or of 4 (2), or none (0).
__device__ __forceinline__ void load8(const LinRows& r, int64_t at, int d0, float* f) {
  LinRaw<kTwo> w{};
  if (r.vec == 2) {
    const char* p = static_cast<const char*>(r.p) + (at + d0) * lin_size(r.type);
    const bool second = d0 + 4 < r.cols;
    if (r.type == 0) {
      w.a = *reinterpret_cast<const u32x4*>(p);
      if (second) w.b = *reinterpret_cast<const u32x4*>(p + 16);
    } else {
      const u32x2 lo = *reinterpret_cast<const u32x2*>(p);
      u32x2 hi = {0, 0};
      if (second) hi = *reinterpret_cast<const u32x2*>(p + 8);
      w.a = u32x4{lo[0], lo[1], hi[0], hi[1]};
    }
  } else {
    w = lin_load8<kTwo>(r, at, d0);
  }
  lin_unpack8<kTwo>(w, r.type, f);
}
__device__ __forceinline__ void store8(const LinRows& r, int64_t at, int d0, const float* f) {
  if (!r.vec) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (d0 + k < r.cols) lin_set<kTwo>(r, at + d0 + k, f[k]);
    return;
  }
  const bool second = r.vec == 1 || d0 + 4 < r.cols;
  char* p = static_cast<char*>(r.p) + (at + d0) * lin_size(r.type);
  if (r.type == 0) {
    *reinterpret_cast<f32x4*>(p) = f32x4{f[0], f[1], f[2], f[3]};
    if (second) *reinterpret_cast<f32x4*>(p + 16) = f32x4{f[4], f[5], f[6], f[7]};
    return;
  }
  u32x4 w;
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = r.type == 1 ? F16::pack2(f[2 * k], f[2 * k + 1]) : BF16::pack2(f[2 * k], f[2 * k + 1]);
  if (r.vec == 1) {
    *reinterpret_cast<u32x4*>(p) = w;
  } else {
    *reinterpret_cast<u32x2*>(p) = u32x2{w[0], w[1]};
    if (second) *reinterpret_cast<u32x2*>(p + 8) = u32x2{w[2], w[3]};
  }
}

// LPR lanes for a row.  A workgroup has p.per rows of a head (rows: batch x n).
template <int LPR, bool BWD>
__global__ __launch_bounds__(kThreads) void gated_norm_kernel(GatedNormParams p) {
  constexpr int kRows = kThreads / LPR;
  __shared__ float red[BWD ? kThreads * 8 : 1];
  const int tid = threadIdx.x, d0 = tid % LPR * 8, r0 = tid / LPR, h = blockIdx.y;
  const int cols = p.x.cols;
  const bool on = d0 < cols;
  const int64_t rows = (int64_t)p.B * p.N, first = (int64_t)blockIdx.x * p.per;
  float w[8], dw[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) w[k] = p.weight && d0 + k < cols ? lin_value(p.weight, p.w_type, h * p.w_sh + d0 + k) : 1.f, dw[k] = 0.f;
  const float inv = 1.f / cols;
  for (int i = r0; i < p.per; i += kRows) {
    const int64_t row = first + i;
    if (row >= rows) break;   // a row's lanes leave together
    const int64_t b = row / p.N, n = row - b * p.N;
    const auto off = [&](const LinRows& r) { return b * r.s[0] + h * r.s[1] + n * r.s[2]; };
    float x[8], g[8], y[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = g[k] = y[k] = 0.f;
    if (on) {
      load8(p.x, off(p.x), d0, x);
      load8(p.gate, off(p.gate), d0, g);
      if (BWD) load8(p.y, off(p.y), d0, y);
    }
    float sg[8], ss = 0.f, tx = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      sg[k] = sigmoid_f(g[k]);
      ss = fmaf(x[k], x[k], ss);
    }
    float t[8];
    if (BWD)
#pragma unroll
      for (int k = 0; k < 8; ++k) t[k] = y[k] * w[k] * g[k] * sg[k], tx = fmaf(t[k], x[k], tx);
#pragma unroll
    for (int m = 1; m < LPR; m *= 2) {
      ss += wave_shfl_xor(ss, m);
      if (BWD) tx += wave_shfl_xor(tx, m);
    }
    float scale = 1.f, eps = p.eps;
    if (!(ss <= kF32Max)) {   // the same of the row at a smaller scale; infinities and NaN stay what they are
      POPE_COLD_PATH();
      scale = kNormDown, eps = ss = tx = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        x[k] *= scale;
        ss = fmaf(x[k], x[k], ss);
        if (BWD) tx = fmaf(t[k], x[k], tx);
      }
#pragma unroll
      for (int m = 1; m < LPR; m *= 2) {
        ss += wave_shfl_xor(ss, m);
        if (BWD) tx += wave_shfl_xor(tx, m);
      }
    }
    const float r = 1.f / __builtin_sqrtf(fmaf(ss, inv, eps));
    if (!on) continue;
    if (!BWD) {
#pragma unroll
      for (int k = 0; k < 8; ++k) y[k] = x[k] * r * w[k] * g[k] * sg[k];
      store8(p.y, off(p.y), d0, y);
    } else {
      const float back = r * r * tx * inv;
      float dx[8], dg[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float xr = x[k] * r;
        dx[k] = r * scale * (t[k] - x[k] * back);
        dg[k] = y[k] * xr * w[k] * sg[k] * fmaf(g[k], 1.f - sg[k], 1.f);
        dw[k] = fmaf(y[k] * xr, g[k] * sg[k], dw[k]);
      }
      store8(p.dx, off(p.dx), d0, dx);
      store8(p.dgate, off(p.dgate), d0, dg);
    }
  }
  if (BWD && p.part) {
#pragma unroll
    for (int k = 0; k < 8; ++k) red[k * kThreads + tid] = dw[k];
    __syncthreads();
    for (int d = tid; d < cols; d += kThreads) {
      float s = 0.f;
      for (int r = 0; r < kRows; ++r) s += red[d % 8 * kThreads + r * LPR + d / 8];
      p.part[((int64_t)h * gridDim.x + blockIdx.x) * cols + d] = s;
    }
  }
}

// dweight: the workgroups' sums, of a head or of all.
constexpr int kSumThreads = 1024;
__global__ __launch_bounds__(kSumThreads) void gated_norm_weight_kernel(GatedNormParams p, int per_head) {
  __shared__ float red[kSumThreads];
  const int tid = threadIdx.x, lane = tid & 63, q = tid >> 6, d = blockIdx.x * 64 + lane, hw = blockIdx.y;
  const int n = p.heads_w == 1 ? p.H * per_head : per_head;
  const float* src = p.part + (p.heads_w == 1 ? 0 : (int64_t)hw * per_head * p.x.cols);
  float s = 0.f;
  if (d < p.x.cols)
#pragma unroll 8
    for (int i = q; i < n; i += kSumThreads / 64) s += src[(int64_t)i * p.x.cols + d];
  red[tid] = s;
  __syncthreads();
  if (q || d >= p.x.cols) return;
  for (int i = 1; i < kSumThreads / 64; ++i) s += red[64 * i + lane];
  const int64_t at = (int64_t)hw * p.x.cols + d;
  if (p.w_type == 0) static_cast<float*>(p.dweight)[at] = s;
  else static_cast<uint16_t*>(p.dweight)[at] = p.w_type == 1 ? F16::bits(s) : BF16::bits(s);
}

// Rows of a head per workgroup: as many workgroups as fill the chip, of at least kNormRows turns.
int rows_per(int64_t rows, int H, int at_once) {
  const int64_t grid = std::max<int64_t>(1, kNormGrid / H), least = (int64_t)at_once * kNormRows;
  return (int)std::min<int64_t>(std::max<int64_t>(least, (rows + grid - 1) / grid), (int64_t)1 << 30);
}
int lanes_per(int cols) { return cols <= 64 ? 8 : cols <= 128 ? 16 : cols <= 256 ? 32 : 64; }

template <bool BWD>
hipError_t norm_t(GatedNormParams p, hipStream_t s) {
  const int lpr = lanes_per(p.x.cols);
  const int64_t rows = (int64_t)p.B * p.N;
  p.per = rows_per(rows, p.H, kThreads / lpr);
  const dim3 grid((unsigned)((rows + p.per - 1) / p.per), p.H), block(kThreads);
  const char* name = BWD ? "gated_norm_bwd" : "gated_norm";
  hipError_t e = lpr == 8 ? launch_named(name, gated_norm_kernel<8, BWD>, grid, block, s, p)
                 : lpr == 16 ? launch_named(name, gated_norm_kernel<16, BWD>, grid, block, s, p)
                 : lpr == 32 ? launch_named(name, gated_norm_kernel<32, BWD>, grid, block, s, p)
                             : launch_named(name, gated_norm_kernel<64, BWD>, grid, block, s, p);
  if (e != hipSuccess || !BWD || !p.part) return e;
  return launch_named("gated_norm_weight", gated_norm_weight_kernel, dim3((p.x.cols + 63) / 64, p.heads_w), dim3(kSumThreads), s, p, (int)grid.x);
}

}  // namespace

int gated_norm_parts(int B, int H, int N, int cols) {
  const int64_t rows = (int64_t)B * N, per = rows_per(rows, H, kThreads / lanes_per(cols));
  return (int)((rows + per - 1) / per) * H;
}

hipError_t launch_gated_norm(const GatedNormParams& p, bool bwd, hipStream_t s) { return bwd ? norm_t<true>(p, s) : norm_t<false>(p, s); }

}  // namespace pope
