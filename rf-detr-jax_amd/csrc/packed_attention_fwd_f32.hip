// packed_attention_fwd_f32.hip — the packed-sequence attention's forward kernels for f32 tensors.
#include "packed_attention_launch.h"

namespace msda_host {
template int dispatch_pk_fwd<float>(const msda::PackParams&, hipStream_t);
}  // namespace msda_host
