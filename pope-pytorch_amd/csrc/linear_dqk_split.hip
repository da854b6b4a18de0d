// Linear attention of rows as sums of two bf16 parts: gradients of the queries and keys.
#include "linear_out.hpp"

namespace pope {

hipError_t launch_linear_dqk_split(const LinOutParams& p, hipStream_t s) { return launch_linear_out_t<kTwo, kLinDq>(p, "linear_dqk", s); }

}  // namespace pope
