// Sliding-window attention for f16 operands.
#include "bkcore_attention_impl.h"

namespace bk {
template void attn_forward<f16_t>(const AttnArgs &, int, bool, hipStream_t);
template void attn_backward<f16_t>(const AttnArgs &, int, bool, hipStream_t);
template void attn_step<f16_t>(const StepArgs &, int, bool, hipStream_t);
}  // namespace bk
