// Linear attention of bf16 rows: gradients of the queries and keys.
#include "linear_out.hpp"

namespace pope {

hipError_t launch_linear_dqk_bf16(const LinOutParams& p, hipStream_t s) { return launch_linear_out_t<kOne, kLinDq>(p, "linear_dqk", s); }

}  // namespace pope
