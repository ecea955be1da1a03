// The launches of the attention's gradient for bfloat16 operands.
#include "attention_gradient_kernel.hpp"

namespace zcgvs_hip {
template int launchAttentionGradient<__bf16>(const AttentionGradientPlan&, const AttentionArgs&, const AttentionGradient&, hipStream_t);
}  // namespace zcgvs_hip
