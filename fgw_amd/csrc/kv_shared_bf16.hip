// Instantiations of kv_extend.h for both passes over shared prefixes, BF16.
#include "kv_extend.h"

namespace fgw_kv {
template hipError_t launch_extend_rows<true, 32, PrefixParams>(const PrefixParams&, int, hipStream_t);
template hipError_t launch_extend_rows<true, 64, PrefixParams>(const PrefixParams&, int, hipStream_t);
template hipError_t launch_extend_rows<true, 128, PrefixParams>(const PrefixParams&, int, hipStream_t);
template hipError_t launch_extend_rows<true, 256, PrefixParams>(const PrefixParams&, int, hipStream_t);
template hipError_t launch_extend_rows<true, 32, SuffixParams>(const SuffixParams&, int, hipStream_t);
template hipError_t launch_extend_rows<true, 64, SuffixParams>(const SuffixParams&, int, hipStream_t);
template hipError_t launch_extend_rows<true, 128, SuffixParams>(const SuffixParams&, int, hipStream_t);
template hipError_t launch_extend_rows<true, 256, SuffixParams>(const SuffixParams&, int, hipStream_t);
}  // namespace fgw_kv
