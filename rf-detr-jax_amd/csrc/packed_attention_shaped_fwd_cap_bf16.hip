// packed_attention_shaped_fwd_cap_bf16.hip — the forward kernels of shaped scores with a cap for bf16 tensors.
#define MSDA_PK_INSTANTIATE
#include "packed_attention_launch.h"

namespace msda_host {
MSDA_PK_FWD(msda::bf16_t, 5);
MSDA_PK_FWD(msda::bf16_t, 7);
}  // namespace msda_host
