// cache4_attention_shaped_f32.hip — attention over a cache in 4 bits, f32 queries, scores in ranges, with slopes.
#define MSDA_C4_INSTANTIATE
#include "cache4_launch.h"

namespace msda_host {
MSDA_C4_FWD(float, 4);
MSDA_C4_FWD(float, 6);
}  // namespace msda_host
