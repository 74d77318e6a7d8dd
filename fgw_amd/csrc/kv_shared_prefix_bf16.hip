// Instantiations of kv_extend_wide.h for the first pass over shared prefixes, BF16.
#include "kv_extend_wide.h"

namespace fgw_kv {
template hipError_t launch_extend_wide<true, 64, PrefixParams>(const PrefixParams&, int, hipStream_t);
template hipError_t launch_extend_wide<true, 128, PrefixParams>(const PrefixParams&, int, hipStream_t);
template hipError_t launch_extend_wide<true, 256, PrefixParams>(const PrefixParams&, int, hipStream_t);
}  // namespace fgw_kv
