// The books of the pages on the device (include/fgw_kv.h), for the kernels that change them: scans over one
// workgroup, the free pages in order, checks.
#pragma once
#include "kv_common.h"

namespace fgw_kv {

typedef uint32_t u32;
typedef int i32x4 __attribute__((ext_vector_type(4), aligned(4)));  // (books may start anywhere)

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;
constexpr int kSlabPer = 16;                          // pages of a thread and step
constexpr int kSlab = kPlanThreads * kSlabPer;
constexpr int kMaxPages = 1 << 20;

struct Books {
  int32_t* refs;
  int32_t* table;
  int32_t* lens;
  int32_t pages, rows, width, page;
};

// Exclusive sum over the workgroup, and the total in every thread. Two barriers.
template <int THREADS = kPlanThreads>
__device__ __forceinline__ int block_scan(int x, int* lds, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // By DPP within rows of 16 lanes (shifts by 1, 2, 4, 8), then each row's last lane onto those behind it.
  int incl = x;
  incl += __builtin_amdgcn_update_dpp(0, incl, 0x111, 0xf, 0xf, false);
  incl += __builtin_amdgcn_update_dpp(0, incl, 0x112, 0xf, 0xf, false);
  incl += __builtin_amdgcn_update_dpp(0, incl, 0x114, 0xf, 0xf, false);
  incl += __builtin_amdgcn_update_dpp(0, incl, 0x118, 0xf, 0xf, false);
  const int r0 = __builtin_amdgcn_readlane(incl, 15), r1 = __builtin_amdgcn_readlane(incl, 31), r2 = __builtin_amdgcn_readlane(incl, 47);
  incl += (lane >= 16 ? r0 : 0) + (lane >= 32 ? r1 : 0) + (lane >= 48 ? r2 : 0);
  __syncthreads();  // lds of the scan before is no longer read
  if (lane == 63) lds[wave] = incl;
  __syncthreads();
  int before = 0;
  total = 0;
  for (int w = 0; w < THREADS / 64; ++w) {
    before += w < wave ? lds[w] : 0;
    total += lds[w];
  }
  return before + incl - x;
}

// The pages [16 i, 16 i + 16) of thread i in the slab at `base`: bit k set when page base + 16 i +
// k exists and is held.
__device__ __forceinline__ u32 held_bits(const int32_t* refs, int pages, int base) {
  const int first = base + (int)threadIdx.x * kSlabPer;
  u32 bits = 0;
  if (first + kSlabPer <= pages) {
    i32x4 x[kSlabPer / 4];
#pragma unroll
    for (int k = 0; k < kSlabPer / 4; ++k) x[k] = *reinterpret_cast<const i32x4*>(refs + first + 4 * k);
#pragma unroll
    for (int k = 0; k < kSlabPer; ++k) bits |= x[k / 4][k % 4] > 0 ? 1u << k : 0u;
  } else {
    for (int k = 0; first + k < pages; ++k) bits |= refs[first + k] > 0 ? 1u << k : 0u;
  }
  return bits;
}
__device__ __forceinline__ u32 page_bits(int pages, int base) {  // pages that exist
  const int n = pages - (base + (int)threadIdx.x * kSlabPer);
  return n <= 0 ? 0u : n >= kSlabPer ? (1u << kSlabPer) - 1u : (1u << n) - 1u;
}

// The free pages in order of id, up to `want`: list[0 .. want); returns how many there are of them.
// `first`: held_bits at page 0, if the caller has read them ahead.
template <int THREADS = kPlanThreads>
__device__ __forceinline__ int rank_free(const Books& b, int want, int32_t* list, int* lds, const u32* first = nullptr) {
  int found = 0;
  for (int base = 0; base < b.pages && found < want; base += THREADS * kSlabPer) {
    u32 free = ~(first && base == 0 ? *first : held_bits(b.refs, b.pages, base)) & page_bits(b.pages, base);
    int total;
    int rank = found + block_scan<THREADS>(__popc(free), lds, total);
    for (; free && rank < want; free &= free - 1u, ++rank)
      list[rank] = base + (int)threadIdx.x * kSlabPer + __ffs(free) - 1;
    found += total;
  }
  return found < want ? found : want;
}

__device__ __forceinline__ int clamp_len(const Books& b, int len) {
  const int cap = b.width * b.page;
  return len < 0 ? 0 : (len > cap ? cap : len);
}

inline int check_books(const fgw_pages_books* b, Books& out) {
  if (!b || !b->refs || !b->table || !b->lens) return fail(FGW_MHA_EINVAL, "page books are missing");
  if (b->pages <= 0 || b->rows <= 0 || b->width <= 0 || b->page_size <= 0)
    return fail(FGW_MHA_EINVAL, "positive pages, rows, table width and page size required");
  if ((int64_t)b->width * b->page_size > 0x7fffffff)
    return fail(FGW_MHA_EUNSUPPORTED, "table capacity must fit in 31 bits");
  if (b->pages > kMaxPages)
    return fail(FGW_MHA_EUNSUPPORTED, "at most %d pages", kMaxPages);
  out = Books{b->refs, b->table, b->lens, b->pages, b->rows, b->width, b->page_size};
  return FGW_MHA_OK;
}

}  // namespace fgw_kv
