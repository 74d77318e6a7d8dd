// Rows of the cache shortened to the keys that carry the most attention weight (fgw_pages_evict).
//
// Row r, len > keep[r] >= first + recent: each layer and K/V head keeps the positions [0, first) and
// [len - recent, len), and of those between the keep - first - recent with the largest sums (ties: the
// lowest position), in order of position. The row's table changes for all layers and heads at once; which
// position holds which old token is each head's own matter.
//
// The kept tokens go to fresh pages, from the page of token `first` on: whole pages below stay where they
// are, and shared pages need no care, since nothing is written that another row holds. So every copy is
// independent of every other. Two launches for up to kMaxLayers layers:
//   evict_select_kernel  program 0 plans: free pages to rows in order (as a reservation), and the list of
//                        rows that shrink. Beside it one program for each (layer, row, head) finds the
//                        smallest kept sum by counting digits of 11 bits from the top (three passes over
//                        the sums, which stay in registers up to 16384 of them), then writes the kept
//                        positions in order, by counts of each wave's part and one scan over them.
//   evict_move_kernel    K and V, 16 bytes to a lane, read by head and written in whole tokens; the sums, in
//                        place (one program a head: it reads a stretch, then writes it; kept tokens only move
//                        down); the books, with the last layers.
// Program 0 is bound by its chain of reads, the moves by memory.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kv_books.h"

namespace fgw_kv {

typedef u32 u32x4 __attribute__((ext_vector_type(4)));

constexpr int kMaxLayers = 16;           // of one pair of launches
constexpr int kPer = 16;                 // sums of a thread in registers
constexpr int kHeld = kPlanThreads * kPer;
constexpr int kBins = 2048;
constexpr int kMoveThreads = 256;
constexpr int kMoveLoads = 2;            // 16-byte chunks of a thread
constexpr int kMovers = 8192;            // workgroups of a launch that count their work on the device
constexpr int kSumLoads = 8;

struct Layers {
  const float* scores[kMaxLayers];
  char* data[2 * kMaxLayers];  // K of all layers, then V
  int32_t head_bytes[2 * kMaxLayers];
};

// What the plan leaves: rows that shrink, in order, with the work of each; their old lengths and tables.
struct EvictPlan {
  int32_t* count;    // rows that shrink
  int32_t* active;   // [rows] which
  int32_t* base;     // [rows + 1] parts of tokens before, by place in `active`
  int32_t* place;    // [rows] of a row's fresh pages in the list
  int32_t* old_len;  // [rows]
  int32_t* list;     // fresh pages
  int32_t* table;    // [rows, width] as it was
  int32_t* kept;     // [layers, rows, heads, capacity] positions
};

struct EvictArgs {
  Books b;
  const int32_t* keep;
  int32_t first, recent, heads, layers, tokens_part;
  int64_t stride;  // of a head's sums
  int64_t capacity;
  EvictPlan plan;
};

// Whether row r shrinks, if pages are left; `bad`: its count is below what has to stay.
__device__ __forceinline__ bool shrinks(const EvictArgs& a, int r, int& len, int& keep, bool& bad) {
  len = clamp_len(a.b, a.b.lens[r]);
  keep = a.keep[r];
  const bool wanted = keep >= 0 && keep < len;
  bad = wanted && (int64_t)a.first + a.recent > keep;
  return wanted && !bad;
}

__device__ __forceinline__ void plan_rows(const EvictArgs& a, int32_t* status) {
  __shared__ int lds[kPlanWaves];
  __shared__ int short_rows, bad_rows;
  const Books& b = a.b;
  if (threadIdx.x == 0) short_rows = bad_rows = 0;
  const int still = a.first / b.page;
  int want = 0;
  for (int base = 0; base < b.rows; base += kPlanThreads) {
    const int r = base + (int)threadIdx.x;
    int len = 0, keep = 0;
    bool bad = false;
    const bool ok = r < b.rows && shrinks(a, r, len, keep, bad);
    const int need = ok ? (int)(((int64_t)keep + b.page - 1) / b.page) - still : 0;
    int total;
    const int before = want + block_scan(need > b.pages ? b.pages + 1 : need, lds, total);
    if (r < b.rows) {
      a.plan.place[r] = before;
      a.plan.old_len[r] = ok ? len : -1;
    }
    if (bad) atomicAdd(&bad_rows, 1);
    want = want + total > b.pages ? b.pages + 1 : want + total;
  }
  const int found = rank_free(b, want < b.pages ? want : b.pages, a.plan.list, lds);
  int count = 0, parts = 0;
  for (int base = 0; base < b.rows; base += kPlanThreads) {
    const int r = base + (int)threadIdx.x;
    bool go = false;
    int part = 0;
    if (r < b.rows && a.plan.old_len[r] >= 0) {
      const int keep = a.keep[r], at = a.plan.place[r];
      const int need = (int)(((int64_t)keep + b.page - 1) / b.page) - still;
      go = need <= 0 || (at <= found && need <= found - at);
      if (!go) atomicAdd(&short_rows, 1);
      part = go ? (keep - still * b.page + a.tokens_part - 1) / a.tokens_part : 0;
    }
    int rows_here, parts_here;
    const int rank = count + block_scan(go ? 1 : 0, lds, rows_here);
    const int before = parts + block_scan(part, lds, parts_here);
    if (go) {
      a.plan.active[rank] = r;
      a.plan.base[rank] = before;
    }
    count += rows_here;
    parts += parts_here;
  }
  // Fresh pages that no refused row stands in front of: held from now on.
  __threadfence_block();
  __syncthreads();
  for (int i = threadIdx.x; i < count; i += kPlanThreads) {
    const int r = a.plan.active[i], at = a.plan.place[r];
    const int need = (int)(((int64_t)a.keep[r] + b.page - 1) / b.page) - still;
    for (int k = 0; k < need; ++k) b.refs[a.plan.list[at + k]] = 1;
  }
  if (threadIdx.x == 0) {
    *a.plan.count = count;
    a.plan.base[count] = parts;
    if (status) {
      status[0] = short_rows;
      status[1] = bad_rows;
    }
  }
}

// Sums in descending order as unsigned numbers; NaN as minus infinity, -0 as 0.
__device__ __forceinline__ u32 sort_key(float x) {
  x = x == x ? x + 0.0f : -INFINITY;
  const u32 u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// blockIdx.x 0: the plan (status: in the call's first launch; else none). Others: one (layer, row, head).
__global__ __launch_bounds__(kPlanThreads) void evict_select_kernel(EvictArgs a, Layers layers, int32_t* status, int plan) {
  __shared__ int lds[kPlanWaves], bins[kBins], picked[2];
  __shared__ int counts[kPer * kPlanWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (blockIdx.x == 0) {
    if (plan) plan_rows(a, status);
    return;
  }
  const int w = (int)blockIdx.x - 1, head = w % a.heads, rest = w / a.heads, r = rest % a.b.rows, layer = rest / a.b.rows;
  int len, keep;
  bool bad;
  if (!shrinks(a, r, len, keep, bad)) return;
  if (plan && layer == 0 && head == 0) {
    const int live = (int)(((int64_t)len + a.b.page - 1) / a.b.page);
    for (int j = tid; j < live; j += kPlanThreads) a.plan.table[(int64_t)r * a.b.width + j] = a.b.table[(int64_t)r * a.b.width + j];
  }
  const int n = len - a.first - a.recent, want = keep - a.first - a.recent;
  const float* const x = layers.scores[layer] + ((int64_t)r * a.heads + head) * a.stride + a.first;
  int32_t* const kept = a.plan.kept + (((int64_t)layer * a.b.rows + r) * a.heads + head) * a.capacity + a.first;
  if (want == 0) return;
  u32 held[kPer];
  auto load = [&](int base) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int i = base + k * kPlanThreads + tid;
      held[k] = i < n ? sort_key(x[i]) : 0u;  // (no sum's key is 0: that of minus infinity is 0x007fffff)
    }
  };
  // The digits of the want-th largest key, from the top.
  u32 prefix = 0;
  int left = want;
  if (n <= kHeld) load(0);
  constexpr int kShift[3] = {21, 10, 0}, kBits[3] = {11, 11, 10};
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    for (int i = tid; i < kBins; i += kPlanThreads) bins[i] = 0;
    __syncthreads();
    for (int base = 0; base < n; base += kHeld) {
      if (n > kHeld) load(base);
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        const bool in = held[k] != 0u && (pass == 0 || held[k] >> (kShift[pass] + kBits[pass]) == prefix);
        if (in) atomicAdd(&bins[held[k] >> kShift[pass] & ((1u << kBits[pass]) - 1u)], 1);
      }
    }
    __syncthreads();
    const int hi = bins[kBins - 1 - 2 * tid], lo = bins[kBins - 2 - 2 * tid];
    int total;
    const int before = block_scan(hi + lo, lds, total);
    if (before < left && left <= before + hi + lo) {
      const bool upper = left <= before + hi;
      picked[0] = kBins - (upper ? 1 : 2) - 2 * tid;
      picked[1] = left - before - (upper ? 0 : hi);
    }
    __syncthreads();
    prefix = prefix << kBits[pass] | (u32)picked[0];
    left = picked[1];
  }
  // All keys above `prefix` and the first `left` of those that equal it, by position.
  int above_before = 0, equal_before = 0;
  for (int base = 0; base < n; base += kHeld) {
    if (n > kHeld) load(base);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int above = __popcll(__ballot(held[k] > prefix)), equal = __popcll(__ballot(held[k] == prefix));
      if (lane == 0) counts[k * kPlanWaves + wave] = above | equal << 16;
    }
    __syncthreads();
    int total;
    const int mine = tid < kPer * kPlanWaves ? counts[tid] : 0;
    const int sum = block_scan(mine, lds, total);  // (at most 16384 of each kind: no carry from the low half)
    if (tid < kPer * kPlanWaves) counts[tid] = sum;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const bool above = held[k] > prefix, equal = held[k] == prefix;
      const uint64_t below = (1ull << lane) - 1ull;
      const int c = counts[k * kPlanWaves + wave];
      const int na = above_before + (c & 0xffff) + __popcll(__ballot(above) & below);
      const int ne = equal_before + (c >> 16) + __popcll(__ballot(equal) & below);
      if (above || (equal && ne < left)) kept[na + (ne < left ? ne : left)] = a.first + base + k * kPlanThreads + tid;
    }
    above_before += total & 0xffff;
    equal_before += total >> 16;
  }
}

// The old position of the token that position d of a row gets, d < keep.
__device__ __forceinline__ int source(const EvictArgs& a, const int32_t* kept, int d, int keep, int len) {
  return d < a.first ? d : d >= keep - a.recent ? d + (len - keep) : kept[d];
}

// blockIdx.y < 2 layers: K or V of a layer, blockIdx.x over parts of tokens; < 3 layers: a layer's sums, over
// (row, head); then the books, over rows.
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictArgs a, Layers layers) {
  const Books& b = a.b;
  const int tid = threadIdx.x, lane = tid & 63, count = *a.plan.count, page = b.page, still = a.first / page;
  const int y = (int)blockIdx.y;
  if (y < 2 * a.layers) {
    const int head_bytes = layers.head_bytes[y], token_bytes = a.heads * head_bytes, layer = y < a.layers ? y : y - a.layers;
    char* const pool = layers.data[y];
    const int chunks = head_bytes / 16, per_token = token_bytes / 16, parts = a.plan.base[count];
    for (int w = blockIdx.x; w < parts; w += gridDim.x) {
      // The row: the last one whose parts begin at w or before.
      int at = 0;
      for (int base = 0; base < count; base += 64) {
        const int mine = base + lane < count ? a.plan.base[base + lane] : 0x7fffffff;
        const int n = __popcll(__ballot(mine <= w));
        if (n > 0) at = base + n - 1;
        if (n < 64) break;
      }
      const int r = a.plan.active[at], len = a.plan.old_len[r], keep = a.keep[r];
      const int d0 = still * page + (w - a.plan.base[at]) * a.tokens_part;
      const int tokens = keep - d0 < a.tokens_part ? keep - d0 : a.tokens_part;
      const int32_t* const old_table = a.plan.table + (int64_t)r * b.width;
      const int32_t* const fresh = a.plan.list + a.plan.place[r];
      const int32_t* const kept = a.plan.kept + ((int64_t)layer * b.rows + r) * a.heads * a.capacity;
      for (int u0 = 0; u0 < tokens * per_token; u0 += kMoveThreads * kMoveLoads) {
        u32x4 x[kMoveLoads];
        char* to[kMoveLoads];
#pragma unroll
        for (int k = 0; k < kMoveLoads; ++k) {
          const int u = u0 + k * kMoveThreads + tid;
          to[k] = nullptr;
          if (u < tokens * per_token) {
            const int t = (int)((u32)u / (u32)per_token), in_token = u - t * per_token;
            const int head = (int)((u32)in_token / (u32)chunks), d = d0 + t;
            const int s = source(a, kept + (int64_t)head * a.capacity, d, keep, len);
            const int sp = (int)((u32)s / (u32)page), dp = (int)((u32)d / (u32)page);
            const int from = old_table[sp], into = fresh[dp - still];
            if (from >= 0 && from < b.pages) {
              const int64_t row = (int64_t)from * page + (s - sp * page), dst = (int64_t)into * page + (d - dp * page);
              x[k] = *reinterpret_cast<const u32x4*>(pool + row * token_bytes + in_token * 16);
              to[k] = pool + dst * token_bytes + in_token * 16;
            }
          }
        }
#pragma unroll
        for (int k = 0; k < kMoveLoads; ++k)
          if (to[k]) *reinterpret_cast<u32x4*>(to[k]) = x[k];
      }
    }
    return;
  }
  if (y < 3 * a.layers) {
    const int layer = y - 2 * a.layers;
    for (int w = blockIdx.x; w < count * a.heads; w += gridDim.x) {
      const int r = a.plan.active[w / a.heads], head = w % a.heads, len = a.plan.old_len[r], keep = a.keep[r];
      const int64_t place = ((int64_t)layer * b.rows + r) * a.heads + head;
      const int32_t* const kept = a.plan.kept + place * a.capacity;
      float* const row = const_cast<float*>(layers.scores[layer]) + ((int64_t)r * a.heads + head) * a.stride;
      for (int base = a.first; base < keep; base += kMoveThreads * kSumLoads) {
        float x[kSumLoads];
#pragma unroll
        for (int k = 0; k < kSumLoads; ++k) {
          const int d = base + k * kMoveThreads + tid;
          x[k] = d < keep ? row[source(a, kept, d, keep, len)] : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < kSumLoads; ++k) asm volatile("" ::"v"(x[k]));  // read before any wave writes
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kSumLoads; ++k) {
          const int d = base + k * kMoveThreads + tid;
          if (d < keep) row[d] = x[k];
        }
      }
    }
    return;
  }
  for (int w = blockIdx.x; w < count; w += gridDim.x) {
    const int r = a.plan.active[w], len = a.plan.old_len[r], keep = a.keep[r];
    const int live = (int)(((int64_t)len + page - 1) / page), pages = (int)(((int64_t)keep + page - 1) / page);
    const int32_t* const fresh = a.plan.list + a.plan.place[r];
    int32_t* const row = b.table + (int64_t)r * b.width;
    for (int j = still + tid; j < b.width; j += kMoveThreads) {
      const int id = row[j];
      if (j < live && id >= 0 && id < b.pages) atomicSub(&b.refs[id], 1);
      row[j] = j < pages ? fresh[j - still] : -1;
    }
    if (tid == 0) b.lens[r] = keep;
  }
}

static int64_t layers_of_launch(int64_t rows, int64_t heads, int64_t capacity, int64_t layers) {
  // (Kept positions of a launch: below 256 MB where one layer's are.)
  const int64_t fit = std::max<int64_t>(1, ((int64_t)1 << 26) / std::max<int64_t>(1, rows * heads * capacity));
  return std::min<int64_t>(std::min<int64_t>(layers, kMaxLayers), fit);
}

static int check_evict(const fgw_pages_books* books, const fgw_evict_args* a, Books& b) {
  if (int rc = check_books(books, b)) return rc;
  if (!a) return fail(FGW_MHA_EINVAL, "arguments are missing");
  if (a->layers <= 0 || a->heads <= 0) return fail(FGW_MHA_EINVAL, "positive layers and heads required");
  if (a->first < 0 || a->recent < 0) return fail(FGW_MHA_EINVAL, "the tokens that always stay must not be negative");
  if (a->scores_stride < (int64_t)b.width * b.page)
    return fail(FGW_MHA_EINVAL, "the scores must have a place for every key of the table");
  if ((int64_t)b.rows * a->heads > 0x7fffffff / (4 * kMaxLayers)) return fail(FGW_MHA_EUNSUPPORTED, "too many rows for one call");
  return FGW_MHA_OK;
}

}  // namespace fgw_kv

using namespace fgw_kv;

extern "C" {

int64_t fgw_pages_evict_workspace(const fgw_pages_books* books, const fgw_evict_args* args) {
  Books b;
  if (int rc = check_evict(books, args, b)) return rc;
  const int64_t capacity = (int64_t)b.width * b.page;
  return 2 + 4 * (int64_t)b.rows + b.pages + (int64_t)b.rows * b.width +
         layers_of_launch(b.rows, args->heads, capacity, args->layers) * b.rows * args->heads * capacity;
}

int fgw_pages_evict(const fgw_pages_books* books, const fgw_evict_args* args, int32_t* status, int32_t* workspace,
                    hipStream_t stream) {
  Books b;
  if (int rc = check_evict(books, args, b)) return rc;
  const fgw_evict_args& a = *args;
  if (!a.keep || !a.k_pools || !a.v_pools || !a.scores || !a.k_head_bytes || !a.v_head_bytes || !status || !workspace)
    return fail(FGW_MHA_EINVAL, "tensors are missing");
  for (int i = 0; i < a.layers; ++i) {
    if (!a.k_pools[i] || !a.v_pools[i] || !a.scores[i]) return fail(FGW_MHA_EINVAL, "tensors are missing");
    for (const int64_t bytes : {a.k_head_bytes[i], a.v_head_bytes[i]})
      if (bytes <= 0 || bytes % 16 || bytes * a.heads > 0x7fffffff / 64)
        return fail(FGW_MHA_EINVAL, "heads of the pools must be multiples of 16 bytes");
    if (!aligned16(a.k_pools[i]) || !aligned16(a.v_pools[i])) return fail(FGW_MHA_EINVAL, "pools must be 16-byte aligned");
  }
  EvictArgs e = {};
  e.b = b;
  e.keep = a.keep;
  e.first = a.first;
  e.recent = a.recent;
  e.heads = a.heads;
  e.stride = a.scores_stride;
  e.capacity = (int64_t)b.width * b.page;
  // A part fills a workgroup's loads about once.
  const int64_t token_bytes = a.k_head_bytes[0] * a.heads;
  e.tokens_part = (int32_t)std::min<int64_t>(64, std::max<int64_t>(1, kMoveThreads * kMoveLoads * 16 / token_bytes));
  EvictPlan& p = e.plan;
  p.count = workspace;
  p.active = p.count + 1;
  p.base = p.active + b.rows;
  p.place = p.base + b.rows + 1;
  p.old_len = p.place + b.rows;
  p.list = p.old_len + b.rows;
  p.table = p.list + b.pages;
  p.kept = p.table + (int64_t)b.rows * b.width;
  const int step = (int)layers_of_launch(b.rows, a.heads, e.capacity, a.layers);
  for (int done = 0; done < a.layers; done += step) {
    Layers layers = {};
    e.layers = std::min(step, a.layers - done);
    for (int i = 0; i < e.layers; ++i) {
      layers.scores[i] = a.scores[done + i];
      layers.data[i] = static_cast<char*>(a.k_pools[done + i]);
      layers.data[e.layers + i] = static_cast<char*>(a.v_pools[done + i]);
      layers.head_bytes[i] = (int32_t)a.k_head_bytes[done + i];
      layers.head_bytes[e.layers + i] = (int32_t)a.v_head_bytes[done + i];
    }
    evict_select_kernel<<<dim3((unsigned)(1 + e.layers * b.rows * a.heads)), dim3(kPlanThreads), 0, stream>>>(
        e, layers, status, done == 0);
    if (int rc = launched("fgw_pages_evict")) return rc;
    const bool last = done + step >= a.layers;
    const int y = 3 * e.layers + (last ? 1 : 0);
    evict_move_kernel<<<dim3((unsigned)std::max(64, kMovers / y), (unsigned)y), dim3(kMoveThreads), 0, stream>>>(e, layers);
    if (int rc = launched("fgw_pages_evict")) return rc;
  }
  return FGW_MHA_OK;
}

}  // extern "C"
