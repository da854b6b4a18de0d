// Linear attention of rows as sums of two bf16 parts: gradients of the values.
#include "linear_out.hpp"

namespace pope {

hipError_t launch_linear_dv_split(const LinOutParams& p, hipStream_t s) { return launch_linear_out_t<kTwo, kLinDv>(p, "linear_dv", s); }

}  // namespace pope
