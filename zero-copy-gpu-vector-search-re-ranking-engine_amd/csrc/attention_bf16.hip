// The attention's launches for bfloat16 operands.
#include "attention_kernel.hpp"

namespace zcgvs_hip {
template int launchAttention<__bf16>(const AttentionPlan&, const AttentionArgs&, const AttentionOutput&, hipStream_t);
}  // namespace zcgvs_hip
