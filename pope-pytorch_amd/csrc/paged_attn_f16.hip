// Instances of the paged attention: 16-bit pages, fp16 queries.
#include "paged_attn.hpp"

namespace pope {

hipError_t launch_paged_attn_f16(const PagedAttnParams& p, bool few, hipStream_t s) {
  return run_paged_shape<F16, false>(p, few, s);
}

}  // namespace pope
