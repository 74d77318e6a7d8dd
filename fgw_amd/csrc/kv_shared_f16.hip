// Instantiations of kv_extend.h for both passes over shared prefixes, F16.
#include "kv_extend.h"

namespace fgw_kv {
template hipError_t launch_extend_rows<false, 32, PrefixParams>(const PrefixParams&, int, hipStream_t);
template hipError_t launch_extend_rows<false, 64, PrefixParams>(const PrefixParams&, int, hipStream_t);
template hipError_t launch_extend_rows<false, 128, PrefixParams>(const PrefixParams&, int, hipStream_t);
template hipError_t launch_extend_rows<false, 256, PrefixParams>(const PrefixParams&, int, hipStream_t);
template hipError_t launch_extend_rows<false, 32, SuffixParams>(const SuffixParams&, int, hipStream_t);
template hipError_t launch_extend_rows<false, 64, SuffixParams>(const SuffixParams&, int, hipStream_t);
template hipError_t launch_extend_rows<false, 128, SuffixParams>(const SuffixParams&, int, hipStream_t);
template hipError_t launch_extend_rows<false, 256, SuffixParams>(const SuffixParams&, int, hipStream_t);
}  // namespace fgw_kv
