// Instantiations of kv_extend_long.h and kv_extend_wide.h for the first pass over shared prefixes, BF16.
#include "kv_extend_long.h"
#include "kv_extend_wide.h"

namespace fgw_kv {
template hipError_t launch_extend_long<true, 64, fgw_mha::kRowsBlock, PrefixParams>(const PrefixParams&, int, hipStream_t);
template hipError_t launch_extend_long<true, 64, fgw_mha::kRowsGroup, PrefixParams>(const PrefixParams&, int, hipStream_t);
template hipError_t launch_extend_long<true, 64, fgw_mha::kRowsPadded, PrefixParams>(const PrefixParams&, int, hipStream_t);
template hipError_t launch_extend_long<true, 128, fgw_mha::kRowsBlock, PrefixParams>(const PrefixParams&, int, hipStream_t);
template hipError_t launch_extend_long<true, 128, fgw_mha::kRowsGroup, PrefixParams>(const PrefixParams&, int, hipStream_t);
template hipError_t launch_extend_long<true, 128, fgw_mha::kRowsPadded, PrefixParams>(const PrefixParams&, int, hipStream_t);
template hipError_t launch_extend_wide<true, 64, PrefixParams>(const PrefixParams&, int, hipStream_t);
template hipError_t launch_extend_wide<true, 128, PrefixParams>(const PrefixParams&, int, hipStream_t);
template hipError_t launch_extend_wide<true, 256, PrefixParams>(const PrefixParams&, int, hipStream_t);
}  // namespace fgw_kv
