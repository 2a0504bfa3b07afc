// packed_attention_shaped_bwd_cap_f32.hip — the backward kernels of shaped scores with a cap for f32 tensors.
#define MSDA_PK_INSTANTIATE
#include "packed_attention_launch.h"

namespace msda_host {
MSDA_PK_BWD(float, 5);
MSDA_PK_BWD(float, 7);
}  // namespace msda_host
