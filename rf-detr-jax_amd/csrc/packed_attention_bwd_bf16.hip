// packed_attention_bwd_bf16.hip — the packed-sequence attention's backward kernels for bf16 tensors.
#include "packed_attention_launch.h"

namespace msda_host {
template int dispatch_pk_bwd<msda::bf16_t>(const msda::PackParams&, int, int, hipStream_t);
}  // namespace msda_host
