// The linear attention's kernels for one type.
#include "decay_kernels.h"

namespace atlhip {

template <>
void decay_fwd<bf16_t>(const DecayGeo& d, const DecayFwd& a, hipStream_t stream) { run_fwd<bf16_t>(d, a, stream); }
template <>
void decay_bwd<bf16_t>(const DecayGeo& d, const DecayBwd& a, hipStream_t stream) { run_bwd<bf16_t>(d, a, stream); }
template <>
void decay_step<bf16_t>(const DecayStep& a, hipStream_t stream) { run_step<bf16_t>(a, stream); }

}  // namespace atlhip
