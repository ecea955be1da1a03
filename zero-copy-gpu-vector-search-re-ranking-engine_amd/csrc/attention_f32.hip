// The attention's launches for float32 operands.
#include "attention_kernel.hpp"

namespace zcgvs_hip {
template int launchAttention<float>(const AttentionPlan&, const AttentionArgs&, const AttentionOutput&, hipStream_t);
}  // namespace zcgvs_hip
