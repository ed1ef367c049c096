// attention_f32.hip -- the forward and dq kernels of attention_tiles.h over float32 elements
#include "attention_tiles.h"

namespace hsgk {
HSGK_ATTN(attn_f32) { return attn_type<float, false>(pass, a, shape, s); }
}  // namespace hsgk
