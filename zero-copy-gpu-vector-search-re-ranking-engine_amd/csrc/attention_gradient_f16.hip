// The launches of the attention's gradient for float16 operands.
#include "attention_gradient_kernel.hpp"

namespace zcgvs_hip {
template int launchAttentionGradient<_Float16>(const AttentionGradientPlan&, const AttentionArgs&, const AttentionGradient&, hipStream_t);
}  // namespace zcgvs_hip
