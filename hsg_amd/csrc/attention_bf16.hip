// attention_bf16.hip -- the forward and dq kernels of attention_tiles.h over bfloat16 elements
#include "attention_tiles.h"

namespace hsgk {
HSGK_ATTN(attn_bf16) { return attn_type<__bf16, false>(pass, a, shape, s); }
}  // namespace hsgk
