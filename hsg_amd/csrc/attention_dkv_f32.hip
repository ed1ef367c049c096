// attention_dkv_f32.hip -- the dk / dv kernels of attention_tiles.h over float32 elements
#include "attention_tiles.h"

namespace hsgk {
HSGK_ATTN(attn_dkv_f32) { return attn_type<float, true>(pass, a, shape, s); }
}  // namespace hsgk
