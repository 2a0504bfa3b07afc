// packed_attention_fwd_bf16.hip — the packed-sequence attention's forward kernels for bf16 tensors.
#include "packed_attention_launch.h"

namespace msda_host {
template int dispatch_pk_fwd<msda::bf16_t>(const msda::PackParams&, hipStream_t);
}  // namespace msda_host
