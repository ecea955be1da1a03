// The linear projection's launches for bfloat16 operands.
#include "linear_kernel.hpp"

namespace zcgvs_hip {
template int launchLinear<__bf16>(const LinearPlan&, int, LinearArgs, hipStream_t);
template int launchLinearSlope<__bf16>(const LinearPlan&, int, LinearArgs, hipStream_t);
template int launchLinearProducts<__bf16>(ProductPlan, bool, ProductArgs, ProductPlan, bool, ProductArgs,
                                          ColumnJoin, hipStream_t);
}  // namespace zcgvs_hip
