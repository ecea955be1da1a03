// The linear projection's launches for int8 operands.
#include "linear_kernel.hpp"

namespace zcgvs_hip {
template int launchLinear<std::int8_t>(const LinearPlan&, int, LinearArgs, hipStream_t);
}  // namespace zcgvs_hip
