// One token of the linear attention for each of many sequences (gfx950): S' = g S + k_hat v^T, o = scale S'^T q_hat, and
// behind it, where there is a gate, o / rms(o) w silu(gate).
//
// Bound by HBM: a state is read and written once (8 E Dv bytes for each sequence and kv head), everything else is a few
// rows.  A workgroup has a state, or, where there are few of them, some of its columns; a thread four columns of every n-th row,
// eight rows in flight.  States, sums and the expanded rows are fp32.
// 200 sequences of 8 kv heads, D 128, R 64, Dv 128: 72 us, 4.5 TB/s (a copy of 1 GiB: 4.9); 64 of 16 heads, D 64, R 64, gated: 17.5, 3.9 TB/s.
#include "linear_dev.hpp"

namespace pope {

namespace {

constexpr int kThreads = 256, kAhead = 8, kMaxE = 512, kMaxDv = 256;

// GM query heads of the key head at once.  MORE: there are others, for which a thread goes over its part of the state again: over
// what it has written, or, where that went nowhere, over what it read.
template <int GM, bool MORE>
__global__ __launch_bounds__(kThreads) void linear_step_kernel(LinStepParams p) {
  __shared__ float kh[kMaxE];
  __shared__ __attribute__((aligned(16))) float qh[GM][kMaxE];
  __shared__ __attribute__((aligned(16))) float part[kThreads * 4];
  __shared__ float out[kMaxDv];
  const LinCall& c = p.c;
  const int tid = threadIdx.x;
  const int wg = blockIdx.x, sp = wg % p.split, rest = wg / p.split, hk = rest % c.Hk, b = rest / c.Hk;
  const int E = c.E, Dv = c.Dv, R = c.R;
  const int from = p.read ? p.read[b] : b, to = p.write ? p.write[b] : from;
  const bool some = (unsigned)from < (unsigned)p.slots;   // no state: no token
  const int cols = ((Dv + p.split - 1) / p.split + 3) & ~3, c0 = sp * cols, c1 = min(Dv, c0 + cols);
  if (c0 >= Dv) return;
  const int across = (c1 - c0 + 3) / 4, groups = kThreads / across;   // threads across a row, rows at once
  const int x4 = tid % across, r0 = tid / across, d0 = c0 + 4 * x4;
  const bool on = r0 < groups;
  const bool vec = Dv % 4 == 0 && p.slot_s % 4 == 0 && (((uintptr_t)p.from | (uintptr_t)p.to) & 15) == 0;
  const float decay = lin_power(lin_log2(c, hk), 1);
  const float* src = p.from + (int64_t)(some ? from : 0) * p.slot_s + (int64_t)hk * E * Dv;
  float* dst = p.to + (int64_t)to * p.slot_s + (int64_t)hk * E * Dv;
  const bool store = some && (unsigned)to < (unsigned)p.slots;

  const auto expand = [&](const LinRows& rows, int h, bool key, float factor, float* to_lds) {
    const int64_t x = (int64_t)b * rows.s[0] + (int64_t)h * rows.s[1];
    for (int d = tid; d < c.D; d += kThreads) {
      const float v = lin_get<kTwo>(rows, x + d);
      if (d < R) {
        float sn, cs;
        sincos_turns(lin_angle_row(c, b, 0)[d], key ? lin_turns(lin_bias(c, hk, d)) : 0.f, &sn, &cs);
        const float m = softplus_f(v) * factor;
        to_lds[2 * d] = m * cs;
        to_lds[2 * d + 1] = m * sn;
      } else {
        to_lds[R + d] = v * factor;
      }
    }
  };
  expand(c.k, hk, true, 1.f, kh);
  float v[4];
#pragma unroll
  for (int r = 0; r < 4; ++r)
    v[r] = on && d0 + r < Dv ? lin_get<kTwo>(c.v, (int64_t)b * c.v.s[0] + (int64_t)hk * c.v.s[1] + d0 + r) : 0.f;

  for (int g0 = 0; g0 < c.G; g0 += GM) {
    const bool again = MORE && g0 && store;   // the new state, from where it went
    const float* in = again ? dst : src;
    if (MORE && g0) __syncthreads();
#pragma unroll
    for (int g = 0; g < GM; ++g)
      if (g0 + g < c.G) expand(c.q, (g0 + g) * c.Hk + hk, false, c.scale, qh[g]);
    __syncthreads();
    f32x4 o[GM];
#pragma unroll
    for (int g = 0; g < GM; ++g) o[g] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (on && some) {
      for (int e0 = r0; e0 < E; e0 += groups * kAhead) {
        f32x4 s[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const int e = e0 + k * groups;
          s[k] = f32x4{0.f, 0.f, 0.f, 0.f};
          if (e >= E) continue;
          if (vec) {
            s[k] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(in + (int64_t)e * Dv + d0));
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (d0 + r < c1) s[k][r] = in[(int64_t)e * Dv + d0 + r];
          }
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const int e = e0 + k * groups;
          if (e >= E) continue;
          if (!again) {
#pragma unroll
            for (int r = 0; r < 4; ++r) s[k][r] = fmaf(kh[e], v[r], decay * s[k][r]);
            if (store) {
              if (vec) __builtin_nontemporal_store(s[k], reinterpret_cast<f32x4*>(dst + (int64_t)e * Dv + d0));
              else
#pragma unroll
                for (int r = 0; r < 4; ++r)
                  if (d0 + r < c1) dst[(int64_t)e * Dv + d0 + r] = s[k][r];
            }
          }
#pragma unroll
          for (int g = 0; g < GM; ++g)
            if (g0 + g < c.G)
#pragma unroll
              for (int r = 0; r < 4; ++r) o[g][r] = fmaf(qh[g][e], s[k][r], o[g][r]);
        }
      }
    }
    // the rows' sums joined, in a fixed order
#pragma unroll
    for (int g = 0; g < GM; ++g) {
      if (g0 + g >= c.G) break;
      __syncthreads();
      if (on) *reinterpret_cast<f32x4*>(part + 4 * tid) = o[g];
      __syncthreads();
      const int h = (g0 + g) * c.Hk + hk;
      if (tid < 4 * across) {
        float sum = 0.f;
        for (int r = 0; r < groups; ++r) sum += part[4 * (r * across) + tid];
        out[tid] = sum;
      }
      const int64_t orow = (int64_t)b * p.o.s[0] + (int64_t)h * p.o.s[1];
      if (!p.gate.p) {
        if (c0 + tid < c1) lin_set<kTwo>(p.o, orow + c0 + tid, out[tid]);
      } else {   // the whole row is here
        __syncthreads();
        if (tid < 64) {
          const auto squares = [&](float scale) {
            float ss = 0.f;
            for (int d = tid; d < Dv; d += 64) ss += (scale * out[d]) * (scale * out[d]);
#pragma unroll
            for (int i = 1; i < 64; i *= 2) ss += wave_shfl_xor(ss, i);
            return ss;
          };
          float down = 1.f, eps = p.eps, ss = squares(1.f);
          if (!(ss <= kF32Max)) down = kNormDown, eps = 0.f, ss = squares(kNormDown);
          const float r = 1.f / __builtin_sqrtf(ss / Dv + eps);
          for (int d = tid; d < Dv; d += 64) {
            const float w = p.weight ? lin_value(p.weight, p.w_type, h * p.w_sh + d) : 1.f;
            const float x = lin_get<kTwo>(p.gate, (int64_t)b * p.gate.s[0] + (int64_t)h * p.gate.s[1] + d);
            lin_set<kTwo>(p.o, orow + d, some ? down * out[d] * r * w * x * sigmoid_f(x) : 0.f);
          }
        }
      }
    }
  }
}

template <int GM, bool MORE>
hipError_t launch(const LinStepParams& p, hipStream_t s) {
  const int64_t n = (int64_t)p.c.seqs.B * p.c.Hk * p.split;
  if (n >= ((int64_t)1 << 22)) return hipErrorInvalidValue;
  return launch_named("linear_step", linear_step_kernel<GM, MORE>, dim3((unsigned)n), dim3(kThreads), s, p);
}

}  // namespace

hipError_t launch_linear_step(const LinStepParams& p, hipStream_t s) {
  const int G = p.c.G;
  return G == 1 ? launch<1, false>(p, s) : G == 2 ? launch<2, false>(p, s) : G <= 4 ? launch<4, false>(p, s) : launch<4, true>(p, s);
}

}  // namespace pope
