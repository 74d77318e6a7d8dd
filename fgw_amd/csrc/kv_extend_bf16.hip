// Instantiations of kv_extend.h, BF16.
#include "kv_extend.h"

namespace fgw_kv {
template hipError_t launch_extend_rows<true, 32, ExtendParams>(const ExtendParams&, int, hipStream_t);
template hipError_t launch_extend_rows<true, 64, ExtendParams>(const ExtendParams&, int, hipStream_t);
template hipError_t launch_extend_rows<true, 128, ExtendParams>(const ExtendParams&, int, hipStream_t);
template hipError_t launch_extend_rows<true, 256, ExtendParams>(const ExtendParams&, int, hipStream_t);
}  // namespace fgw_kv
