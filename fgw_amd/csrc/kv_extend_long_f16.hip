// Instantiations of kv_extend_long.h, F16.
#include "kv_extend_long.h"

namespace fgw_kv {
template hipError_t launch_extend_long<false, 64, fgw_mha::kRowsBlock>(const ExtendParams&, int, hipStream_t);
template hipError_t launch_extend_long<false, 64, fgw_mha::kRowsGroup>(const ExtendParams&, int, hipStream_t);
template hipError_t launch_extend_long<false, 64, fgw_mha::kRowsPadded>(const ExtendParams&, int, hipStream_t);
template hipError_t launch_extend_long<false, 128, fgw_mha::kRowsBlock>(const ExtendParams&, int, hipStream_t);
template hipError_t launch_extend_long<false, 128, fgw_mha::kRowsGroup>(const ExtendParams&, int, hipStream_t);
template hipError_t launch_extend_long<false, 128, fgw_mha::kRowsPadded>(const ExtendParams&, int, hipStream_t);
}  // namespace fgw_kv
