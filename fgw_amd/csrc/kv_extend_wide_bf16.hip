// Instantiation of kv_extend_wide.h, BF16.
#include "kv_extend_wide.h"

namespace fgw_kv {
template hipError_t launch_extend_wide<true, 256, ExtendParams>(const ExtendParams&, int, hipStream_t);
}  // namespace fgw_kv
