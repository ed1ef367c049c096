// attention_dkv_bf16.hip -- the dk / dv kernels of attention_tiles.h over bfloat16 elements
#include "attention_tiles.h"

namespace hsgk {
HSGK_ATTN(attn_dkv_bf16) { return attn_type<__bf16, true>(pass, a, shape, s); }
}  // namespace hsgk
