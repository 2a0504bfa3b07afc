// cache4_attention_plain_f32.hip — attention over a cache in 4 bits, f32 queries, scores without a shape.
#define MSDA_C4_INSTANTIATE
#include "cache4_launch.h"

namespace msda_host {
MSDA_C4_FWD(float, 0);
}  // namespace msda_host
