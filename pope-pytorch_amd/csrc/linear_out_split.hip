// Linear attention of rows as sums of two bf16 parts: outputs.
#include "linear_out.hpp"

namespace pope {

hipError_t launch_linear_out_split(const LinOutParams& p, hipStream_t s) { return launch_linear_out_t<kTwo, kLinOut>(p, "linear_out", s); }

}  // namespace pope
