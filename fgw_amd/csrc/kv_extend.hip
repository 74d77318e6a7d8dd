// C ABI of the attention over pages with grouped heads. The kernels stand in kv_extend.h,
// kv_extend_long.h and kv_extend_wide.h, their instantiations in the kv_extend_*.hip files of each type,
// the choice among them in kv_extend_plan.h.
#include <hip/hip_runtime.h>

#include "kv_extend_plan.h"

namespace fgw_kv {

#define FGW_KV_EXTERN_LONG(BF, DP)                                                                    \
  extern template hipError_t launch_extend_long<BF, DP, kRowsBlock, ExtendParams>(const ExtendParams&, int, hipStream_t); \
  extern template hipError_t launch_extend_long<BF, DP, kRowsGroup, ExtendParams>(const ExtendParams&, int, hipStream_t); \
  extern template hipError_t launch_extend_long<BF, DP, kRowsPadded, ExtendParams>(const ExtendParams&, int, hipStream_t);
extern template hipError_t launch_extend_wide<true, 256, ExtendParams>(const ExtendParams&, int, hipStream_t);
extern template hipError_t launch_extend_wide<false, 256, ExtendParams>(const ExtendParams&, int, hipStream_t);
FGW_KV_EXTERN_LONG(true, 64) FGW_KV_EXTERN_LONG(true, 128)
FGW_KV_EXTERN_LONG(false, 64) FGW_KV_EXTERN_LONG(false, 128)

#define FGW_KV_EXTERN_ROWS(BF, DP) \
  extern template hipError_t launch_extend_rows<BF, DP, ExtendParams>(const ExtendParams&, int, hipStream_t);
FGW_KV_EXTERN_ROWS(true, 32) FGW_KV_EXTERN_ROWS(true, 64)
FGW_KV_EXTERN_ROWS(true, 128) FGW_KV_EXTERN_ROWS(true, 256)
FGW_KV_EXTERN_ROWS(false, 32) FGW_KV_EXTERN_ROWS(false, 64)
FGW_KV_EXTERN_ROWS(false, 128) FGW_KV_EXTERN_ROWS(false, 256)

}  // namespace fgw_kv

using namespace fgw_kv;

extern "C" {

int fgw_kv_extend_workspace(const fgw_kv_extend_args* args, int64_t* floats, int64_t* counters) {
  if (int rc = check(args)) return rc;
  *floats = *counters = 0;
  if (args->tokens == 0) return FGW_MHA_OK;
  const Plan l = plan(*args);
  *floats = l.rows.floats + l.longs.floats;
  *counters = l.rows.counters;
  return FGW_MHA_OK;
}

int fgw_kv_extend(const fgw_kv_extend_args* args, hipStream_t stream) {
  if (int rc = check(args)) return rc;
  const fgw_kv_extend_args& a = *args;
  if (a.tokens == 0) return FGW_MHA_OK;
  if (int rc = check_tensors(a)) return rc;
  const Plan l = plan(a);
  if (std::max(l.rows.items, l.longs.items) > 0x3fffffff)
    return fail(FGW_MHA_EUNSUPPORTED, "too many rows for one call");
  if (l.rows.floats + l.longs.floats > 0 && (!a.workspace || !aligned16(a.workspace)))
    return fail(FGW_MHA_EINVAL, "the workspace is missing");
  ExtendParams p = params_of<ExtendParams>(a);
  p.parts = a.workspace;
  p.counters = l.rows.counters > 0 ? a.counters : nullptr;
  return a.dtype == FGW_KV_BFLOAT16 ? run<true>(p, l, "fgw_kv_extend", stream)
                                    : run<false>(p, l, "fgw_kv_extend", stream);
}

}  // extern "C"
