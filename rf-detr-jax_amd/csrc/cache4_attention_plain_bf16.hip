// cache4_attention_plain_bf16.hip — attention over a cache in 4 bits, bf16 queries, scores without a shape.
#define MSDA_C4_INSTANTIATE
#include "cache4_launch.h"

namespace msda_host {
MSDA_C4_FWD(msda::bf16_t, 0);
}  // namespace msda_host
