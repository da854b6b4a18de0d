// Parameter blocks and launchers of the paged cache's kernels, shared with the C ABI.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "paged_index.hpp"
#include "pope_kernels.hpp"

namespace pope {

// The cache and the call's view of it.
struct PagedCache {
  void* k; void* v; uint8_t* scales;   // pages; scales: 8-bit caches only
  const int* table; int64_t table_sb;  // (B, columns) page numbers
  PagedSeqs seqs;
  int pages, blk_shift;                // blocks per page: 1 << blk_shift
  int Hk, D, R, steps, tiles;          // tiles: V tiles of 16 columns (PagedSeqs knows the rows)
  int64_t k_head, v_head;              // elements of one (page, head)
};

struct PagedRowsParams {               // write: k, v -> cache; read: cache -> k, v
  PagedCache c;
  void* k; void* v;                    // rows (b, h, n); read: k rows of D + R columns
  const float* freqs; const float* bias;
  int64_t k_s[3], v_s[3], f_s[2], bias_sh;
  int k_vec, v_vec, f_vec;             // rows of whole 16-byte units (f: of angles and bias)
  int64_t blocks;                      // grid.x: blocks of 32 slots over all sequences
};
hipError_t launch_paged_write(const PagedRowsParams& p, int dtype, bool q8, hipStream_t s);
hipError_t launch_paged_read(const PagedRowsParams& p, int dtype, bool q8, hipStream_t s);

struct PagedAttnParams {
  PagedCache c;
  const uint16_t* q; const float* freqs;
  uint16_t* o; float* lse;             // lse may be null: (batch, Hq, rows) natural log
  PagedDiv G;                          // Hq / Hk
  int Hq, causal, N;                   // N: rows per batch entry (all of them when packed)
  int splits, least;                   // splits of the key axis, the least blocks of one (few rows: paged_few_least)
  int slots;                           // workgroups that the chip holds: paged_plan raises `least` (many rows); 0: `least` stands
  int64_t tiles;                       // row tiles
  // Scores come out of the products in log2 units: Q_hat carries q_factor = softmax scale x log2 e.  fp16 does not hold
  // every Q_hat times a factor above 1: the scores then take `late`, the factor's magnitude, and q_factor its sign.
  float q_factor, late;
  int64_t q_s[3], o_s[3], f_s[2];
  int q_vec, f_vec, o_vec;             // query rows: whole 16-byte units; angles likewise; output rows: 8-byte units
  float* part_o; float* part_ml;       // splits > 1: (tile, head, row, split): 16 * tiles floats, and (m, l)
  int* parts;                          // splits > 1: (tile, head): splits that have keys
};
// Rows of a tile: 16 where a sequence has at most as many (query head of a key head, new token) rows on average, else 128.
constexpr int kPagedFewRows = 16, kPagedManyRows = 128;
hipError_t launch_paged_attn(const PagedAttnParams& p, bool few, int dtype, bool q8, hipStream_t s);

// One translation unit each (paged_attn_*.hip).
hipError_t launch_paged_attn_bf16(const PagedAttnParams& p, bool few, hipStream_t s);
hipError_t launch_paged_attn_f16(const PagedAttnParams& p, bool few, hipStream_t s);
hipError_t launch_paged_attn_bf16_8(const PagedAttnParams& p, bool few, hipStream_t s);
hipError_t launch_paged_attn_f16_8(const PagedAttnParams& p, bool few, hipStream_t s);

}  // namespace pope
