// Sliding-window attention for bf16 operands.
#include "bkcore_attention_impl.h"

namespace bk {
template void attn_forward<bf16_t>(const AttnArgs &, int, bool, hipStream_t);
template void attn_backward<bf16_t>(const AttnArgs &, int, bool, hipStream_t);
template void attn_step<bf16_t>(const StepArgs &, int, bool, hipStream_t);
}  // namespace bk
