// Instances of the paged attention: 16-bit pages, bf16 queries.
#include "paged_attn.hpp"

namespace pope {

hipError_t launch_paged_attn_bf16(const PagedAttnParams& p, bool few, hipStream_t s) {
  return run_paged_shape<BF16, false>(p, few, s);
}

}  // namespace pope
