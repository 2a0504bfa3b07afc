// cache4_attention_cap_bf16.hip — attention over a cache in 4 bits, bf16 queries, scores with a cap.
#define MSDA_C4_INSTANTIATE
#include "cache4_launch.h"

namespace msda_host {
MSDA_C4_FWD(msda::bf16_t, 5);
MSDA_C4_FWD(msda::bf16_t, 7);
}  // namespace msda_host
