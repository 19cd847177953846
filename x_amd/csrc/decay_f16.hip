// The linear attention's kernels for one type.
#include "decay_kernels.h"

namespace atlhip {

template <>
void decay_fwd<f16_t>(const DecayGeo& d, const DecayFwd& a, hipStream_t stream) { run_fwd<f16_t>(d, a, stream); }
template <>
void decay_bwd<f16_t>(const DecayGeo& d, const DecayBwd& a, hipStream_t stream) { run_bwd<f16_t>(d, a, stream); }
template <>
void decay_step<f16_t>(const DecayStep& a, hipStream_t stream) { run_step<f16_t>(a, stream); }

}  // namespace atlhip
