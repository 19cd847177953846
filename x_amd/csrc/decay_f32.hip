// The linear attention's kernels for one type.
#include "decay_kernels.h"

namespace atlhip {

template <>
void decay_fwd<float>(const DecayGeo& d, const DecayFwd& a, hipStream_t stream) { run_fwd<float>(d, a, stream); }
template <>
void decay_bwd<float>(const DecayGeo& d, const DecayBwd& a, hipStream_t stream) { run_bwd<float>(d, a, stream); }
template <>
void decay_step<float>(const DecayStep& a, hipStream_t stream) { run_step<float>(a, stream); }

}  // namespace atlhip
