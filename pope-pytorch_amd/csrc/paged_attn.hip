// Dispatch of the paged attention to its instances (paged_attn_*.hip).
#include "paged.hpp"

namespace pope {

hipError_t launch_paged_attn(const PagedAttnParams& p, bool few, int dtype, bool q8, hipStream_t s) {
  if (dtype == 2) return q8 ? launch_paged_attn_bf16_8(p, few, s) : launch_paged_attn_bf16(p, few, s);
  return q8 ? launch_paged_attn_f16_8(p, few, s) : launch_paged_attn_f16(p, few, s);
}

}  // namespace pope
