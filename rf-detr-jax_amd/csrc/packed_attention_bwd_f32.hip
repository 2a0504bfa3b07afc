// packed_attention_bwd_f32.hip — the packed-sequence attention's backward kernels for f32 tensors.
#define MSDA_PK_INSTANTIATE
#include "packed_attention_launch.h"

namespace msda_host {
MSDA_PK_BWD(float, 0);
}  // namespace msda_host
