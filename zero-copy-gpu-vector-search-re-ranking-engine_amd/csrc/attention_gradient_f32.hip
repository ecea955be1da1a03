// The launches of the attention's gradient for float32 operands.
#include "attention_gradient_kernel.hpp"

namespace zcgvs_hip {
template int launchAttentionGradient<float>(const AttentionGradientPlan&, const AttentionArgs&, const AttentionGradient&, hipStream_t);
}  // namespace zcgvs_hip
