// packed_attention_fwd_bf16.hip — the packed-sequence attention's forward kernels for bf16 tensors.
#define MSDA_PK_INSTANTIATE
#include "packed_attention_launch.h"

namespace msda_host {
MSDA_PK_FWD(msda::bf16_t, 0);
}  // namespace msda_host
