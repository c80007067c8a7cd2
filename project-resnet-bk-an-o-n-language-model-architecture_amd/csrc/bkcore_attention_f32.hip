// Sliding-window attention for f32 operands.
#include "bkcore_attention_impl.h"

namespace bk {
template void attn_forward<float>(const AttnArgs &, int, bool, hipStream_t);
template void attn_backward<float>(const AttnArgs &, int, bool, hipStream_t);
template void attn_step<float>(const StepArgs &, int, bool, hipStream_t);
}  // namespace bk
