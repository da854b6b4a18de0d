// Dispatch of the paged attention to its instances (paged_attn_*.hip).
#include "paged.hpp"

namespace pope {

// Few rows: one tile of 16 (or 32) rows that all four waves share, over the blocks of keys.  Many: 4 x 32 rows, each wave
// with rows of its own over all keys; 4 x 16 rows where the row is so wide (V tiles of 16 columns: 16) that two
// column tiles leave the registers.
PagedPlan paged_plan(int64_t rows, int tiles) {
  if (rows <= 16) return {1, 4};
  if (tiles > 8) return rows <= 32 ? PagedPlan{1, 4} : PagedPlan{1, 1};
  return rows <= 64 ? PagedPlan{2, 4} : PagedPlan{2, 1};
}

hipError_t launch_paged_attn(const PagedAttnParams& p, PagedPlan plan, int dtype, bool q8, hipStream_t s) {
  if (dtype == 2) return q8 ? launch_paged_attn_bf16_8(p, plan, s) : launch_paged_attn_bf16(p, plan, s);
  return q8 ? launch_paged_attn_f16_8(p, plan, s) : launch_paged_attn_f16(p, plan, s);
}

}  // namespace pope
