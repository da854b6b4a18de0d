// Instances of the paged attention: 8-bit pages, bf16 queries.
#include "paged_attn.hpp"

namespace pope {

hipError_t launch_paged_attn_bf16_8(const PagedAttnParams& p, bool few, hipStream_t s) {
  return run_paged_shape<BF16, true>(p, few, s);
}

}  // namespace pope
