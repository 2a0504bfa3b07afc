// cache4_attention_cap_f32.hip — attention over a cache in 4 bits, f32 queries, scores with a cap.
#define MSDA_C4_INSTANTIATE
#include "cache4_launch.h"

namespace msda_host {
MSDA_C4_FWD(float, 5);
MSDA_C4_FWD(float, 7);
}  // namespace msda_host
