// packed_attention_shaped_fwd_f32.hip — the forward kernels of shaped scores without a cap for f32 tensors.
#define MSDA_PK_INSTANTIATE
#include "packed_attention_launch.h"

namespace msda_host {
MSDA_PK_FWD(float, 4);
MSDA_PK_FWD(float, 6);
}  // namespace msda_host
