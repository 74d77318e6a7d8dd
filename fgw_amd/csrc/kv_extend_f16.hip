// Instantiations of kv_extend.h, F16.
#include "kv_extend.h"

namespace fgw_kv {
template hipError_t launch_extend_rows<false, 32, ExtendParams>(const ExtendParams&, int, hipStream_t);
template hipError_t launch_extend_rows<false, 64, ExtendParams>(const ExtendParams&, int, hipStream_t);
template hipError_t launch_extend_rows<false, 128, ExtendParams>(const ExtendParams&, int, hipStream_t);
template hipError_t launch_extend_rows<false, 256, ExtendParams>(const ExtendParams&, int, hipStream_t);
}  // namespace fgw_kv
