// Linear attention of fp16 rows: outputs.
#include "linear_out.hpp"

namespace pope {

hipError_t launch_linear_out_f16(const LinOutParams& p, hipStream_t s) { return launch_linear_out_t<F16, kLinOut>(p, "linear_out", s); }

}  // namespace pope
