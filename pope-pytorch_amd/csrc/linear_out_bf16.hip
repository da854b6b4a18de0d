// Linear attention of bf16 rows: outputs.
#include "linear_out.hpp"

namespace pope {

hipError_t launch_linear_out_bf16(const LinOutParams& p, hipStream_t s) { return launch_linear_out_t<kOne, kLinOut>(p, "linear_out", s); }

}  // namespace pope
