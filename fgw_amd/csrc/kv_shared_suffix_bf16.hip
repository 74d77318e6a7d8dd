// Instantiations of kv_extend_long.h and kv_extend_wide.h for the second pass over shared prefixes, BF16.
#include "kv_extend_long.h"
#include "kv_extend_wide.h"

namespace fgw_kv {
template hipError_t launch_extend_long<true, 64, fgw_mha::kRowsBlock, SuffixParams>(const SuffixParams&, int, hipStream_t);
template hipError_t launch_extend_long<true, 64, fgw_mha::kRowsGroup, SuffixParams>(const SuffixParams&, int, hipStream_t);
template hipError_t launch_extend_long<true, 64, fgw_mha::kRowsPadded, SuffixParams>(const SuffixParams&, int, hipStream_t);
template hipError_t launch_extend_long<true, 128, fgw_mha::kRowsBlock, SuffixParams>(const SuffixParams&, int, hipStream_t);
template hipError_t launch_extend_long<true, 128, fgw_mha::kRowsGroup, SuffixParams>(const SuffixParams&, int, hipStream_t);
template hipError_t launch_extend_long<true, 128, fgw_mha::kRowsPadded, SuffixParams>(const SuffixParams&, int, hipStream_t);
template hipError_t launch_extend_wide<true, 256, SuffixParams>(const SuffixParams&, int, hipStream_t);
}  // namespace fgw_kv
