// attention_f16.hip -- the forward and dq kernels of attention_tiles.h over float16 elements
#include "attention_tiles.h"

namespace hsgk {
HSGK_ATTN(attn_f16) { return attn_type<_Float16, false>(pass, a, shape, s); }
}  // namespace hsgk
