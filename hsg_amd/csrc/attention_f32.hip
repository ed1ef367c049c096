// attention_f32.hip -- the attention kernels (attention_tiles.h) over fp32 elements; one type a file so that they build
// side by side
#include "attention_tiles.h"

namespace hsgk {
int attn_f32(AttnPass pass, const AttnArgs &a, bool wk, hipStream_t s) { return attn_type<float>(pass, a, wk, s); }
}  // namespace hsgk
