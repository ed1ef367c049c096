// attention_bf16.hip -- the attention kernels (attention_tiles.h) over bfloat16 elements; one type a file so that they build
// side by side
#include "attention_tiles.h"

namespace hsgk {
int attn_bf16(AttnPass pass, const AttnArgs &a, bool wk, hipStream_t s) { return attn_type<__bf16>(pass, a, wk, s); }
}  // namespace hsgk
