// What the sources behind include/fgw_kv.h share: the error message of the calling thread, the
// checks' shorthand and small device helpers.
#pragma once
#include <hip/hip_runtime.h>

#include <stdint.h>

#include "../../include/fgw_kv.h"

namespace fgw_kv {

// Records the message of a failure and returns its status.
int fail(int status, const char* format, ...) __attribute__((format(printf, 2, 3)));
// FGW_MHA_OK, or the error that the last launch left.
int launched(const char* what);

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Multiplier and shift of fgw_mha::div_page for a page size.
inline void page_division(uint32_t page, uint32_t& magic, uint32_t& shift) {
  shift = 0;
  while ((1ull << shift) < page) ++shift;
  magic = (uint32_t)((((uint64_t)1 << 32) * ((1ull << shift) - page)) / page + 1);
}

}  // namespace fgw_kv
