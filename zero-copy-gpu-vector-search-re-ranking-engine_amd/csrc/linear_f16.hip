// The linear projection's launches for float16 operands.
#include "linear_kernel.hpp"

namespace zcgvs_hip {
template int launchLinear<_Float16>(const LinearPlan&, int, LinearArgs, hipStream_t);
template int launchLinearSlope<_Float16>(const LinearPlan&, int, LinearArgs, hipStream_t);
template int launchLinearProducts<_Float16>(ProductPlan, bool, ProductArgs, ProductPlan, bool, ProductArgs,
                                          ColumnJoin, hipStream_t);
}  // namespace zcgvs_hip
