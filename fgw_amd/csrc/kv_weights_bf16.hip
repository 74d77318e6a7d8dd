// Instantiations of kv_weights.h, BF16.
#include "kv_weights.h"

namespace fgw_kv {
template hipError_t launch_weights<true, 64>(const WeightParams&, bool, int, hipStream_t);
template hipError_t launch_weights<true, 128>(const WeightParams&, bool, int, hipStream_t);
template hipError_t launch_weights<true, 256>(const WeightParams&, bool, int, hipStream_t);
template hipError_t launch_weights_columns<true, 64>(const WeightParams&, int, hipStream_t);
template hipError_t launch_weights_columns<true, 128>(const WeightParams&, int, hipStream_t);
template hipError_t launch_weights_columns<true, 256>(const WeightParams&, int, hipStream_t);
}  // namespace fgw_kv
