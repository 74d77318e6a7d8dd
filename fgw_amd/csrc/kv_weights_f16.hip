// Instantiations of kv_weights.h, F16.
#include "kv_weights.h"

namespace fgw_kv {
template hipError_t launch_weights<false, 64>(const WeightParams&, bool, int, hipStream_t);
template hipError_t launch_weights<false, 128>(const WeightParams&, bool, int, hipStream_t);
template hipError_t launch_weights<false, 256>(const WeightParams&, bool, int, hipStream_t);
template hipError_t launch_weights_columns<false, 64>(const WeightParams&, int, hipStream_t);
template hipError_t launch_weights_columns<false, 128>(const WeightParams&, int, hipStream_t);
template hipError_t launch_weights_columns<false, 256>(const WeightParams&, int, hipStream_t);
}  // namespace fgw_kv
