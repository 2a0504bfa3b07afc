// cache4_attention_shaped_bf16.hip — attention over a cache in 4 bits, bf16 queries, scores in ranges, with slopes.
#define MSDA_C4_INSTANTIATE
#include "cache4_launch.h"

namespace msda_host {
MSDA_C4_FWD(msda::bf16_t, 4);
MSDA_C4_FWD(msda::bf16_t, 6);
}  // namespace msda_host
