// The linear projection's launches for float32 operands.
#include "linear_kernel.hpp"

namespace zcgvs_hip {
template int launchLinear<float>(const LinearPlan&, int, LinearArgs, hipStream_t);
template int launchLinearSlope<float>(const LinearPlan&, int, LinearArgs, hipStream_t);
template int launchLinearProducts<float>(ProductPlan, bool, ProductArgs, ProductPlan, bool, ProductArgs,
                                          ColumnJoin, hipStream_t);
}  // namespace zcgvs_hip
