// The attention's launches for float16 operands.
#include "attention_kernel.hpp"

namespace zcgvs_hip {
template int launchAttention<_Float16>(const AttentionPlan&, const AttentionArgs&, const AttentionOutput&, hipStream_t);
}  // namespace zcgvs_hip
