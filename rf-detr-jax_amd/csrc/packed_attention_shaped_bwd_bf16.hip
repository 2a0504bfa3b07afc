// packed_attention_shaped_bwd_bf16.hip — the backward kernels of shaped scores without a cap for bf16 tensors.
#define MSDA_PK_INSTANTIATE
#include "packed_attention_launch.h"

namespace msda_host {
MSDA_PK_BWD(msda::bf16_t, 4);
MSDA_PK_BWD(msda::bf16_t, 6);
}  // namespace msda_host
