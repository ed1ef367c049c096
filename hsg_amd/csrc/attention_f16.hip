// attention_f16.hip -- the attention kernels (attention_tiles.h) over float16 elements; one type a file so that they build
// side by side
#include "attention_tiles.h"

namespace hsgk {
int attn_f16(AttnPass pass, const AttnArgs &a, bool wk, hipStream_t s) { return attn_type<_Float16>(pass, a, wk, s); }
}  // namespace hsgk
