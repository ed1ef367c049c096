// attention_dkv_f16.hip -- the dk / dv kernels of attention_tiles.h over float16 elements
#include "attention_tiles.h"

namespace hsgk {
HSGK_ATTN(attn_dkv_f16) { return attn_type<_Float16, true>(pass, a, shape, s); }
}  // namespace hsgk
