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
//                        smallest kept sum by counting digits of 11 bits from the top, until the sums that
//                        share them are few enough to compare with each other (at most three passes over
//                        the sums, which stay in registers up to 16384 of them), then writes the kept
//                        positions in order, by counts of each wave's part and one scan over them.
//   evict_move_kernel    K and V in parts of some tokens: a thread finds the place of one (token, head), then
//                        all copy, 16 bytes to a lane, and write whole tokens; the sums, in place (one program
//                        a head: it reads a stretch, then writes it; kept tokens only move down); the books,
//                        with the last layers.
// Measured (BF16, D 128, 8 K/V heads): 16 rows of up to 4096 keys, 12 of them cut to 1000, four layers: select
// 13 us, as long as a program's chain of passes and scans takes, moves 78 us (profiled), 5.0 TB/s of the 393 MB
// that they read and write, at memory's rate. One row of 381 keys (FP16, D 64) cut to 200: 8 and 6 us, chains of reads.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kv_books.h"

namespace fgw_kv {

typedef u32 u32x4 __attribute__((ext_vector_type(4)));

constexpr int kMaxLayers = 16;           // of one pair of launches
constexpr int kPer = 16;                 // sums of a thread in registers
// Threads of a program where capacities fit its registers (else kPlanThreads): its scans and barriers are those of
// four waves, and eight programs share a CU. 256 / 1024 threads, us of a call: 64 rows of 2048 keys, four layers
// 352 / 400, one row of 1024 16.8 / 19.4.
constexpr int kFewThreads = 256;
// Counters of a bin: lanes with equal sums meet in it. One / four, us of a call that moves nothing: 16 rows of 16384
// equal sums 111 / 50, of 4096 33 / 21, of random ones 15.5 / 17.0.
constexpr int kBins = 2048, kCopies = 4;
// Keys that are compared with each other in place of the passes that are left. With / without, us: 64 rows of 2048
// 352 / 362, one of 1024 16.8 / 19.9.
constexpr int kDirect = 256;
constexpr int kMoveThreads = 256;
constexpr int kMoveLoads = 8;            // 16-byte chunks of a thread at once (4 / 8, us: 64 rows of 2048 383 / 342)
constexpr int kMovers = 4096;            // workgroups of a launch that count their work on the device
constexpr int kSumLoads = 8;
// Tokens of a part: as many as make kPartBytes of K or V, fewer where all rows at their capacity would be less than
// kSpread parts. 8 / 16 / 32 KB, us: 12 of 16 rows to 1000 keys, four layers 111 / 101 / 106, 8 rows of 16384 keys to
// 8000, 4 heads 120 / 106 / 108, 8 heads of D 256 179 / 179 / 183; at least 4 / 16 tokens: one row 15.2 / 17.0.
constexpr int kLeastPart = 4;
constexpr int64_t kPartBytes = 16384;
constexpr int kSpread = 2048;

struct Layers {
  const float* scores[kMaxLayers];
  char* data[2 * kMaxLayers];  // K of all layers, then V
  int32_t head_bytes[2 * kMaxLayers];
};

// A row that shrinks: its number, old length, budget, and where its fresh pages begin in the list.
struct Shrunk {
  int32_t row, len, keep, place;
};
// What the plan leaves.
struct EvictPlan {
  Shrunk* rows;      // [rows], in order
  int32_t* count;    // of them
  int32_t* base;     // [rows + 1] parts of tokens before each, and all parts
  int32_t* need;     // [rows] of rows past the first THREADS
  int32_t* list;     // fresh pages
  int32_t* table;    // [rows, width] as it was
  int32_t* kept;     // [layers, rows, heads, capacity] positions
};

struct EvictArgs {
  Books b;
  const int32_t* keep;
  int32_t first, recent, heads, layers, part;  // tokens of a part
  int64_t stride;                              // of a head's sums
  int64_t capacity;
  EvictPlan plan;
};

// Whether row r shrinks, if pages are left; `bad`: its count is below what has to stay.
__device__ __forceinline__ bool shrinks(const EvictArgs& a, int length, int keep, int& len, bool& bad) {
  len = clamp_len(a.b, length);
  const bool wanted = keep >= 0 && keep < len;
  bad = wanted && (int64_t)a.first + a.recent > keep;
  return wanted && !bad;
}

// Free pages to rows in order, as a reservation does. What a thread knows of its first row stays with it: the
// plan is bound by its round trips to memory.
template <int THREADS>
__device__ __forceinline__ void plan_rows(const EvictArgs& a, int32_t* status) {
  __shared__ int lds[THREADS / 64];
  __shared__ int short_rows, bad_rows, given;
  const Books& b = a.b;
  const int tid = threadIdx.x, still = a.first / b.page;
  if (tid == 0) short_rows = bad_rows = given = 0;
  struct Row {
    int len, keep, need;  // need -1: the row stays
  };
  auto load = [&](int r) {
    Row x{0, -1, -1};
    if (r >= b.rows) return x;
    x.keep = a.keep[r];
    bool bad;
    if (shrinks(a, b.lens[r], x.keep, x.len, bad)) x.need = (int)(((int64_t)x.keep + b.page - 1) / b.page) - still;
    return x;
  };
  const u32 held = held_bits(b.refs, b.pages, 0);  // (beside the lengths)
  const Row mine = load(tid);
  __syncthreads();
  int want = 0, at0 = 0;
  for (int base = 0; base < b.rows; base += THREADS) {
    const Row x = base == 0 ? mine : load(base + tid);
    int total;
    const int need = x.need < 0 ? 0 : (x.need > b.pages ? b.pages + 1 : x.need);
    const int before = want + block_scan<THREADS>(need, lds, total);
    if (base == 0)
      at0 = before;
    else if (base + tid < b.rows)
      a.plan.need[base + tid] = before;
    want = want + total > b.pages ? b.pages + 1 : want + total;
  }
  const int found = rank_free<THREADS>(b, want < b.pages ? want : b.pages, a.plan.list, lds, &held);
  int count = 0, parts = 0;
  for (int base = 0; base < b.rows; base += THREADS) {
    const int r = base + tid;
    const Row x = base == 0 ? mine : load(r);
    const int at = base == 0 ? at0 : (r < b.rows ? a.plan.need[r] : 0);
    const bool go = x.need == 0 || (x.need > 0 && at <= found && x.need <= found - at);
    if (x.need < 0 && x.keep >= 0 && x.keep < x.len) atomicAdd(&bad_rows, 1);  // (it is below what has to stay)
    if (x.need > 0 && !go) atomicAdd(&short_rows, 1);
    if (x.need > 0 && go) atomicMax(&given, at + x.need);
    const int part = go ? (x.keep - still * b.page + a.part - 1) / a.part : 0;
    int rows_here, parts_here;
    const int rank = count + block_scan<THREADS>(go ? 1 : 0, lds, rows_here);
    const int before = parts + block_scan<THREADS>(part, lds, parts_here);
    if (go) {
      a.plan.rows[rank] = Shrunk{r, x.len, x.keep, at};
      a.plan.base[rank] = before;
    }
    count += rows_here;
    parts += parts_here;
  }
  // (Rows in order: the pages that are given are the first ones of the list.)
  __threadfence_block();
  __syncthreads();
  for (int i = tid; i < given; i += THREADS) b.refs[a.plan.list[i]] = 1;
  if (tid == 0) {
    *a.plan.count = count;
    a.plan.base[count] = parts;
    status[0] = short_rows;
    status[1] = bad_rows;
  }
}

// Sums in descending order as unsigned numbers; NaN as minus infinity, -0 as 0.
__device__ __forceinline__ u32 sort_key(float x) {
  x = x == x ? x + 0.0f : -INFINITY;
  const u32 u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// blockIdx.x 0: the plan (in the call's first launch). Others: one (layer, row, head).
template <int THREADS>
__global__ __launch_bounds__(THREADS) void evict_select_kernel(EvictArgs a, Layers layers, int32_t* status, int plan) {
  constexpr int kWaves = THREADS / 64, kHeld = THREADS * kPer;
  __shared__ __attribute__((aligned(16))) int bins[kBins * kCopies];
  __shared__ __attribute__((aligned(16))) u32 few[kDirect];
  __shared__ int lds[kWaves], picked[3], counts[kPer * kWaves], few_count;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (blockIdx.x == 0) {
    if (plan) plan_rows<THREADS>(a, status);
    return;
  }
  const int w = (int)blockIdx.x - 1, head = w % a.heads, rest = w / a.heads, r = rest % a.b.rows, layer = rest / a.b.rows;
  const float* const x = layers.scores[layer] + ((int64_t)r * a.heads + head) * a.stride + a.first;
  const int most = a.capacity > a.first ? (int)a.capacity - a.first : 0;  // sums that there are from `first` on
  const int length = a.b.lens[r], keep = a.keep[r];
  float raw[kPer];
  auto read = [&](int base) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int i = base + k * THREADS + tid;
      raw[k] = i < most ? x[i] : 0.0f;
    }
  };
  if (most <= kHeld) read(0);  // (on the way beside the length)
  int len;
  bool bad;
  if (!shrinks(a, length, keep, len, bad)) return;
  if (plan && layer == 0 && head == 0) {
    const int live = (int)(((int64_t)len + a.b.page - 1) / a.b.page);
    for (int j = tid; j < live; j += THREADS) a.plan.table[(int64_t)r * a.b.width + j] = a.b.table[(int64_t)r * a.b.width + j];
  }
  const int n = len - a.first - a.recent, want = keep - a.first - a.recent;
  int32_t* const kept = a.plan.kept + (((int64_t)layer * a.b.rows + r) * a.heads + head) * a.capacity + a.first;
  if (want == 0) return;
  u32 held[kPer];
  auto load = [&](int base) {
    if (most > kHeld) read(base);
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      held[k] = base + k * THREADS + tid < n ? sort_key(raw[k]) : 0u;  // (no sum's key is 0: that of minus infinity is 0x007fffff)
  };
  // The digits of the want-th largest key, from the top, until the keys that share them are few: those are
  // compared with each other. Lanes take turns at the kCopies counters of a bin, which lie in different banks.
  u32 prefix = 0;
  int left = want;
  const int steps = (n + THREADS - 1) / THREADS < kPer ? (n + THREADS - 1) / THREADS : kPer;
  if (most <= kHeld) load(0);
  bool done = false;
  for (int pass = 0; pass < 3 && !done; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    for (int i = tid; i < kBins * kCopies / 4; i += THREADS) reinterpret_cast<int4*>(bins)[i] = int4{0, 0, 0, 0};
    __syncthreads();
    for (int base = 0; base < n; base += kHeld) {
      if (most > kHeld) load(base);
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        const bool in = k < steps && held[k] != 0u && (pass == 0 || held[k] >> (shift + bits) == prefix);
        if (in) atomicAdd(&bins[(held[k] >> shift & ((1u << bits) - 1u)) * kCopies + (lane & (kCopies - 1))], 1);
      }
    }
    __syncthreads();
    // Each thread has kBins / THREADS bins, from the highest down.
    constexpr int kMine = kBins / THREADS;
    int mine[kMine], sum = 0;
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      const int4 c = reinterpret_cast<const int4*>(bins)[kBins - 1 - (kMine * tid + k)];
      mine[k] = c.x + c.y + c.z + c.w;
      sum += mine[k];
    }
    int total;
    int before = block_scan<THREADS>(sum, lds, total);
    if (before < left && left <= before + sum) {
#pragma unroll
      for (int k = 0; k < kMine; ++k) {
        if (before < left && left <= before + mine[k]) {
          picked[0] = kBins - 1 - (kMine * tid + k);
          picked[1] = left - before;
          picked[2] = mine[k];
        }
        before += mine[k];
      }
    }
    __syncthreads();
    prefix = prefix << bits | (u32)picked[0];
    left = picked[1];
    const int share = picked[2];
    if (pass == 2 || share > kDirect || most > kHeld) continue;
    done = true;
    if (tid == 0) few_count = 0;
    for (int i = tid; i < kDirect; i += THREADS) few[i] = 0u;  // (below every key)
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      if (held[k] != 0u && held[k] >> shift == prefix) few[atomicAdd(&few_count, 1)] = held[k];
    __syncthreads();
    const u32 own = tid < kDirect ? few[tid] : 0u;
    int above = 0, equal = 0;
    for (int i = 0; i < share; i += 4) {
      const uint4 o = *reinterpret_cast<const uint4*>(few + i);
      above += (o.x > own) + (o.y > own) + (o.z > own) + (o.w > own);
      equal += (o.x == own) + (o.y == own) + (o.z == own) + (o.w == own);
    }
    if (own != 0u && above < left && left <= above + equal) {  // (all equal ones write the same)
      picked[0] = (int)own;
      picked[1] = left - above;
    }
    __syncthreads();
    prefix = (u32)picked[0];
    left = picked[1];
  }
  // All keys above `prefix` and the first `left` of those that equal it, by position.
  int above_before = 0, equal_before = 0;
  for (int base = 0; base < n; base += kHeld) {
    if (most > kHeld) load(base);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int above = __popcll(__ballot(held[k] > prefix)), equal = __popcll(__ballot(held[k] == prefix));
      if (lane == 0) counts[k * kWaves + wave] = above | equal << 16;
    }
    __syncthreads();
    int total;
    const int mine = tid < kPer * kWaves ? counts[tid] : 0;
    const int sum = block_scan<THREADS>(mine, lds, total);  // (at most 16384 of each kind: no carry from the low half)
    if (tid < kPer * kWaves) counts[tid] = sum;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      if (k >= steps) continue;
      const bool above = held[k] > prefix, equal = held[k] == prefix;
      const uint64_t below = (1ull << lane) - 1ull;
      const int c = counts[k * kWaves + wave];
      const int na = above_before + (c & 0xffff) + __popcll(__ballot(above) & below);
      const int ne = equal_before + (c >> 16) + __popcll(__ballot(equal) & below);
      if (above || (equal && ne < left)) kept[na + (ne < left ? ne : left)] = a.first + base + k * THREADS + tid;
    }
    above_before += total & 0xffff;
    equal_before += total >> 16;
  }
}

// The old position of the token that position d of a row gets, d < keep.
__device__ __forceinline__ int source(const EvictArgs& a, const int32_t* kept, int d, int keep, int len) {
  return d < a.first ? d : d >= keep - a.recent ? d + (len - keep) : kept[d];
}

// blockIdx.y < layers: K and V of a layer, blockIdx.x over parts of tokens; < 2 layers: a layer's sums, over
// (row, head); then the books, over rows. A part: each thread finds the pool rows of one (token, head), then
// all copy, 16 bytes to a lane, whole tokens written.
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictArgs a, Layers layers) {
  __shared__ int64_t from_row[kMoveThreads], to_row[kMoveThreads];  // of a (token, head), of a token
  const Books& b = a.b;
  const int tid = threadIdx.x, lane = tid & 63, count = *a.plan.count, page = b.page, still = a.first / page;
  const int y = (int)blockIdx.y;
  if (y < a.layers) {
    const int parts = a.plan.base[count];
    for (int w = blockIdx.x; w < parts; w += gridDim.x) {
      // The row: the last one whose parts begin at w or before.
      int at = 0;
      for (int base = 0; base < count; base += 64) {
        const int mine = base + lane < count ? a.plan.base[base + lane] : 0x7fffffff;
        const int n = __popcll(__ballot(mine <= w));
        if (n > 0) at = base + n - 1;
        if (n < 64) break;
      }
      const Shrunk row = a.plan.rows[at];
      const int d0 = still * page + (w - a.plan.base[at]) * a.part, tokens = row.keep - d0 < a.part ? row.keep - d0 : a.part;
      __syncthreads();  // the part before is copied
      {
        const int head = (int)((u32)tid / (u32)a.part), t = tid - head * a.part, d = d0 + t;
        if (head < a.heads && t < tokens) {
          const int32_t* const kept = a.plan.kept + (((int64_t)y * b.rows + row.row) * a.heads + head) * a.capacity;
          const int s = source(a, kept, d, row.keep, row.len), sp = (int)((u32)s / (u32)page);
          const int id = a.plan.table[(int64_t)row.row * b.width + sp];
          from_row[t * a.heads + head] = id >= 0 && id < b.pages ? (int64_t)id * page + (s - sp * page) : -1;
          if (head == 0) {
            const int dp = (int)((u32)d / (u32)page);
            to_row[t] = (int64_t)a.plan.list[row.place + dp - still] * page + (d - dp * page);
          }
        }
      }
      __syncthreads();
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const int which = v ? a.layers + y : y, chunks = layers.head_bytes[which] / 16, per_token = a.heads * chunks;
        char* const pool = layers.data[which];
        const int64_t token_bytes = (int64_t)per_token * 16;
        for (int u0 = 0; u0 < tokens * per_token; u0 += kMoveThreads * kMoveLoads) {
          u32x4 x[kMoveLoads];
          char* to[kMoveLoads];
#pragma unroll
          for (int k = 0; k < kMoveLoads; ++k) {
            const int u = u0 + k * kMoveThreads + tid;
            to[k] = nullptr;
            if (u < tokens * per_token) {
              const int pair = (int)((u32)u / (u32)chunks), t = (int)((u32)pair / (u32)a.heads);
              const int64_t in_token = (int64_t)(u - t * per_token) * 16, from = from_row[pair];
              if (from >= 0) {
                x[k] = *reinterpret_cast<const u32x4*>(pool + from * token_bytes + in_token);
                to[k] = pool + to_row[t] * token_bytes + in_token;
              }
            }
          }
#pragma unroll
          for (int k = 0; k < kMoveLoads; ++k)
            if (to[k]) __builtin_nontemporal_store(x[k], reinterpret_cast<u32x4*>(to[k]));
        }
      }
    }
    return;
  }
  if (y < 2 * a.layers) {
    const int layer = y - a.layers;
    for (int w = blockIdx.x; w < count * a.heads; w += gridDim.x) {
      const Shrunk s = a.plan.rows[w / a.heads];
      const int head = w % a.heads;
      const int64_t place = ((int64_t)layer * b.rows + s.row) * a.heads + head;
      const int32_t* const kept = a.plan.kept + place * a.capacity;
      float* const row = const_cast<float*>(layers.scores[layer]) + ((int64_t)s.row * a.heads + head) * a.stride;
      for (int base = a.first; base < s.keep; base += kMoveThreads * kSumLoads) {
        float x[kSumLoads];
#pragma unroll
        for (int k = 0; k < kSumLoads; ++k) {
          const int d = base + k * kMoveThreads + tid;
          x[k] = d < s.keep ? row[source(a, kept, d, s.keep, s.len)] : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < kSumLoads; ++k) asm volatile("" ::"v"(x[k]));  // read before any wave writes
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kSumLoads; ++k) {
          const int d = base + k * kMoveThreads + tid;
          if (d < s.keep) row[d] = x[k];
        }
      }
      // Tokens of pages outside the pool, which no part copied: zeros, as such pages read to the attention. (Here,
      // since the copies have no registers left for it: 120 of 128.)
      for (int d = still * page + tid; d < s.keep; d += kMoveThreads) {
        const int at = (int)((u32)source(a, kept, d, s.keep, s.len) / (u32)page), id = a.plan.table[(int64_t)s.row * b.width + at];
        if (id >= 0 && id < b.pages) continue;
        const int dp = (int)((u32)d / (u32)page);
        const int64_t token = (int64_t)a.plan.list[s.place + dp - still] * page + (d - dp * page);
#pragma unroll 1
        for (int which = layer; which < 2 * a.layers; which += a.layers) {
          const int64_t bytes = layers.head_bytes[which];
          char* const to = layers.data[which] + (token * a.heads + head) * bytes;
#pragma unroll 1
          for (int64_t c = 0; c < bytes; c += 16) *reinterpret_cast<u32x4*>(to + c) = u32x4{0u, 0u, 0u, 0u};
        }
      }
    }
    return;
  }
  for (int w = blockIdx.x; w < count; w += gridDim.x) {
    const Shrunk s = a.plan.rows[w];
    const int live = (int)(((int64_t)s.len + page - 1) / page), pages = (int)(((int64_t)s.keep + page - 1) / page);
    const int32_t* const fresh = a.plan.list + s.place;
    int32_t* const row = b.table + (int64_t)s.row * b.width;
    for (int j = still + tid; j < b.width; j += kMoveThreads) {
      const int id = row[j];
      if (j < live && id >= 0 && id < b.pages) atomicSub(&b.refs[id], 1);
      row[j] = j < pages ? fresh[j - still] : -1;
    }
    if (tid == 0) b.lens[s.row] = s.keep;
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
  if (a->heads > kMoveThreads) return fail(FGW_MHA_EUNSUPPORTED, "at most %d K/V heads", kMoveThreads);
  if (a->first < 0 || a->recent < 0) return fail(FGW_MHA_EINVAL, "the tokens that always stay must not be negative");
  if ((int64_t)b.width * b.page > 0x7fffffff - 0x10000)  // (positions run on by a program's reads past the last)
    return fail(FGW_MHA_EUNSUPPORTED, "table capacity must fit in 31 bits");
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
  return 8 + 6 * (int64_t)b.rows + b.pages + (int64_t)b.rows * b.width +
         layers_of_launch(b.rows, args->heads, capacity, args->layers) * b.rows * args->heads * capacity;
}

int fgw_pages_evict(const fgw_pages_books* books, const fgw_evict_args* args, int32_t* status, int32_t* workspace,
                    hipStream_t stream) {
  Books b;
  if (int rc = check_evict(books, args, b)) return rc;
  const fgw_evict_args& a = *args;
  if (!aligned16(workspace)) return fail(FGW_MHA_EINVAL, "the workspace must be 16-byte aligned");
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
  // Parts of kPartBytes, with a thread for each (token, head); smaller ones where there are few tokens at most.
  int64_t widest = 0;
  for (int i = 0; i < a.layers; ++i) widest = std::max(widest, std::max(a.k_head_bytes[i], a.v_head_bytes[i]));
  const int64_t tokens = std::max<int64_t>(kPartBytes / (widest * a.heads), kLeastPart);
  const int64_t spread = e.capacity * b.rows * a.layers / kSpread;
  e.part = (int32_t)std::min(std::min<int64_t>(tokens, kMoveThreads / a.heads), std::max<int64_t>(spread, kLeastPart));
  EvictPlan& p = e.plan;
  p.rows = reinterpret_cast<Shrunk*>(workspace);
  p.count = workspace + 4 * (int64_t)b.rows;
  p.base = p.count + 1;
  p.need = p.base + b.rows + 1;
  p.list = p.need + b.rows;
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
    const dim3 programs((unsigned)(1 + e.layers * b.rows * a.heads));
    if (e.capacity <= kFewThreads * kPer)
      evict_select_kernel<kFewThreads><<<programs, dim3(kFewThreads), 0, stream>>>(e, layers, status, done == 0);
    else
      evict_select_kernel<kPlanThreads><<<programs, dim3(kPlanThreads), 0, stream>>>(e, layers, status, done == 0);
    if (int rc = launched("fgw_pages_evict")) return rc;
    const bool last = done + step >= a.layers;
    const int y = 2 * e.layers + (last ? 1 : 0);
    evict_move_kernel<<<dim3((unsigned)std::max(64, kMovers / y), (unsigned)y), dim3(kMoveThreads), 0, stream>>>(e, layers);
    if (int rc = launched("fgw_pages_evict")) return rc;
  }
  return FGW_MHA_OK;
}

}  // extern "C"
