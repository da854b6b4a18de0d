// Parameter blocks and launchers of the linear attention's kernels and of the gated norm, shared with the C ABI.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "linear_rows.hpp"
#include "pope_kernels.hpp"

namespace pope {

// The rows of a call as segments of at most L rows of one sequence.  Padded batches: M segments for each of B sequences.
// Packed rows: a sequence's segments follow those of the sequences before it; T is the most that N rows can have.
struct LinSeqs {
  const int* cu;   // packed: B + 1 bounds
  int B, N, L, M, T;
};

// Expanded rows of one side, bf16: (batch, H, N, EP), columns behind E zeros; the second part, where there is one, `plane`
// elements behind the first.
struct LinHat {
  uint16_t* p;
  int64_t plane;
  int H, EP;
};

struct LinCall {
  LinSeqs seqs;
  LinRows q, k, v, g;            // g: dO
  LinHat qh, kh;                 // queries times the scale; keys that the mask leaves out are zeros
  const float* freqs; int64_t f_s[2]; int f_vec;
  const void* bias; int bias_type; int64_t bias_sh;   // pope_dtype
  const float* log_decay;        // one for each kv head, or null: no decay
  const uint8_t* mask; int64_t mask_sb;
  int Hq, Hk, G, D, R, E, Dv;    // E = D + R
  float scale;
  int split;                     // operands as the sum of two bf16 parts; 0: one part, all rows bf16
};

// What each segment adds to the state behind it (forward), or to the gradient of the state before it (reverse):
// (T, Hk, E, Dv) fp32, rows in the column order of apply_pope_to_qk.
struct LinStateParams {
  LinCall c;
  float* states;                 // launch_linear_states: null for the expanded rows only
  int reverse;
  int tiles, key_wgs, q_parts;   // set by the launchers
};
hipError_t launch_linear_states(const LinStateParams& p, hipStream_t s);   // expands rows; forward: writes them
hipError_t launch_linear_sums(const LinStateParams& p, hipStream_t s);     // from the expanded rows, which are as exact as `split` says

// Those sums to the states that segments start from, in place; `first` (B, Hk, E, Dv) or null: the state before everything
// (reverse: the gradient of the state behind it), `last` or null takes what is left at the other end.
struct LinScanParams {
  LinCall c;
  float* states; const float* first; float* last;
  int reverse;
};
hipError_t launch_linear_scan(const LinScanParams& p, hipStream_t s);

// What a job computes: rows x_i, y_j of P columns and z_j, out_i = sum_{j <= i} g^(i - j) (x_i . y_j) z_j + what the state
// carries in.  Gradients of keys and values go over the rows in reverse.
enum LinKind { kLinOut = 0, kLinDq = 1, kLinDk = 2, kLinDv = 3 };
struct LinOutParams {
  LinCall c;
  LinRows out[2];                // of the launch's kinds: one, or dq and dk
  const float* states[2];        // (T, Hk, E, Dv) that segments start from, forward and reverse; null: `first`
  const float* first[2];         // (B, Hk, E, Dv) or null: zeros
  float* dbias;                  // kLinDk: (T, Hk, R), or null
  float* dphase[2];              // (b, h, n, R) of the kind's rows, or null
  int heads_per;                 // query heads of a key head per workgroup (kLinOut, kLinDq)
  int tiles, first_wgs;          // set by the launchers
};
// One translation unit each.
hipError_t launch_linear_out_bf16(const LinOutParams& p, hipStream_t s);
hipError_t launch_linear_out_split(const LinOutParams& p, hipStream_t s);
hipError_t launch_linear_dqk_bf16(const LinOutParams& p, hipStream_t s);
hipError_t launch_linear_dqk_split(const LinOutParams& p, hipStream_t s);
hipError_t launch_linear_dv_bf16(const LinOutParams& p, hipStream_t s);
hipError_t launch_linear_dv_split(const LinOutParams& p, hipStream_t s);

// dbias (Hb, R) from the segments' parts; dfreqs (Fb, N, R) from the rows' dphase of queries and keys.
struct LinPhaseParams {
  LinCall c;
  const float* part; void* dbias; int Hb;   // dbias in the bias's type
  const float* dphase_q; const float* dphase_k; float* dfreqs; int64_t df_s[2]; int Fb;
};
hipError_t launch_linear_phase(const LinPhaseParams& p, hipStream_t s);

// One token for each of B sequences against its state.
struct LinStepParams {
  LinCall c;
  LinRows o;
  const float* from; float* to;  // (slots, Hk, E, Dv), slots `slot_s` elements apart
  const int* read; const int* write;   // slots of the sequences, or null: their numbers
  int64_t slot_s;
  int slots;
  LinRows gate; const void* weight; int64_t w_sh; int w_type; float eps;   // gate.p null: none
  int split;                     // workgroups for a (sequence, kv head): each has some of the value's columns
};
hipError_t launch_linear_step(const LinStepParams& p, hipStream_t s);

// y = x rsqrt(mean x^2 + eps) w silu(gate) over rows (b, h, n), and its gradients.
struct GatedNormParams {
  LinRows x, gate, y;            // backward: y is dy
  LinRows dx, dgate;
  const void* weight; int64_t w_sh; int w_type;   // (1 or H, cols), null: ones
  float* part;                   // backward: (workgroups, cols) sums of dweight, or null
  void* dweight;                 // (1 or H, cols) in the weight's type
  int B, H, N, heads_w;          // heads_w: rows of the weight
  float eps;
  int per;                       // set by the launcher: rows of a head per workgroup
};
int gated_norm_parts(int B, int H, int N, int cols);   // workgroups of the backward
hipError_t launch_gated_norm(const GatedNormParams& p, bool bwd, hipStream_t s);

}  // namespace pope
