// Linear attention of bf16 rows: gradients of the values.
#include "linear_out.hpp"

namespace pope {

hipError_t launch_linear_dv_bf16(const LinOutParams& p, hipStream_t s) { return launch_linear_out_t<kOne, kLinDv>(p, "linear_dv", s); }

}  // namespace pope
