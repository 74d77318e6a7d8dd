// Errors and version of the C ABI in include/fgw_kv.h; the operators stand in kv_rotary.hip,
// kv_pages.hip and kv_extend.hip.
#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdio>

#include "kv_common.h"

namespace fgw_kv {

static thread_local char g_error[512] = "";

int fail(int status, const char* format, ...) {
  va_list ap;
  va_start(ap, format);
  vsnprintf(g_error, sizeof(g_error), format, ap);
  va_end(ap);
  return status;
}

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? FGW_MHA_OK : fail(FGW_MHA_EHIP, "%s: %s", what, hipGetErrorString(e));
}

}  // namespace fgw_kv

extern "C" {

int fgw_kv_abi_version(void) { return FGW_KV_ABI_VERSION; }

const char* fgw_kv_last_error(void) { return fgw_kv::g_error; }

}  // extern "C"
