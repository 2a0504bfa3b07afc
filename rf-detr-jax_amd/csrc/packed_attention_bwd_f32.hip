// packed_attention_bwd_f32.hip — the packed-sequence attention's backward kernels for f32 tensors.
#include "packed_attention_launch.h"

namespace msda_host {
template int dispatch_pk_bwd<float>(const msda::PackParams&, int, int, hipStream_t);
}  // namespace msda_host
