// Pages of the cache: reserve, fork (copy on write), free, compact and copy (fgw_pages_*).
//
// The books are int32 arrays on the device (include/fgw_kv.h) and every decision is made there, so
// that a serving loop neither waits for the device nor leaves a captured graph. A page is handed
// out by its rank among the free pages in order of id, to rows in order: the same books and pools
// on every run, with atomics only where sums of integers meet.
//
// Two launches: `plan` (one workgroup: scans the holders of all pages, ranks what is free or has to
// move, and writes the books of rows and pages that need no long walk) and `move` (the whole card:
// pools' pages, 16 bytes to a lane, and the rows of the table). The plan is bound by the latency of
// its few dependent reads: every thread takes 16 holders with four independent loads, 16384 pages to
// a step of one scan. A reservation is that plan alone (a call with its launch: 32 rows of 512 pages
// 5.1 us, 256 of 4096 5.6, 1024 of 65536 9.6). The moves are bound by memory: each page read and
// written once in every pool, 32 bytes to a thread (compact 205 pages of 32 KB in 16 pools, fork 40
// of 128 KB in 16, us, 32 / 64 / 128 / 256 bytes: 44 / 46 / 49 / 50, 25.1 / 25.8 / 26.5 / 30). Reads
// go through the caches, since the children of a row copy the same page (40 of 16 rows: 28 us, 44
// with non-temporal reads); what is written is not read soon.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kv_books.h"

namespace fgw_kv {

typedef u32 u32x4 __attribute__((ext_vector_type(4)));

constexpr int kMoveThreads = 256;
constexpr int kMoveLoads = 2;                         // 16-byte chunks of a thread
constexpr int kMovers = 8192;                         // workgroups of moves counted on the device
constexpr int kPart = kMoveThreads * kMoveLoads * 16;  // bytes of a page that one workgroup moves
constexpr int kMaxPools = 64;                         // of one launch

// work: [0, rows] exclusive sums of the rows' needs, then the free pages' list.
__global__ __launch_bounds__(kPlanThreads) void reserve_kernel(Books b, const int32_t* counts,
                                                               int32_t* status, int32_t* work) {
  __shared__ int lds[kPlanWaves];
  __shared__ int short_rows, bad_rows;
  if (threadIdx.x == 0) short_rows = bad_rows = 0;
  int32_t* const first = work;
  int32_t* const list = work + b.rows + 1;
  const int64_t cap = (int64_t)b.width * b.page;
  // Pages that row r needs for counts[r] more tokens (one more than the pool has stands for every
  // number that it cannot meet: the sums stay in 32 bits).
  auto need_of = [&](int r, bool& bad) {
    const int64_t len = b.lens[r], add = counts[r];
    bad = add < 0 || len < 0 || len + add > cap;
    if (bad) return 0;
    const int64_t need = (len + add + b.page - 1) / b.page - (len + b.page - 1) / b.page;
    return (int)(need > b.pages ? b.pages + 1 : need);
  };
  int want = 0;
  for (int base = 0; base < b.rows; base += kPlanThreads) {
    const int r = base + (int)threadIdx.x;
    bool bad = false;
    const int need = r < b.rows ? need_of(r, bad) : 0;
    int total;
    const int before = want + block_scan(need, lds, total);
    if (r < b.rows) first[r] = before;
    if (bad) atomicAdd(&bad_rows, 1);
    want = want + total > b.pages ? b.pages + 1 : want + total;
  }
  const int found = rank_free(b, want < b.pages ? want : b.pages, list, lds);
  __threadfence_block();
  __syncthreads();
  auto granted = [&](int at, int need) { return need == 0 || (at <= found && need <= found - at); };
  // The k-th page goes to the last row whose sum is not above k.
  for (int k = threadIdx.x; k < found; k += kPlanThreads) {
    int lo = 0, hi = b.rows;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first[mid] <= k) lo = mid; else hi = mid;
    }
    bool bad;
    const int need = need_of(lo, bad), at = first[lo];
    if (bad || k - at >= need || !granted(at, need)) continue;
    const int have = (int)(((int64_t)b.lens[lo] + b.page - 1) / b.page);
    const int page = list[k];
    b.table[(int64_t)lo * b.width + have + (k - at)] = page;
    b.refs[page] = 1;
  }
  __syncthreads();
  for (int r = threadIdx.x; r < b.rows; r += kPlanThreads) {
    bool bad;
    const int need = need_of(r, bad);
    if (bad) continue;
    if (granted(first[r], need))
      b.lens[r] += counts[r];
    else
      atomicAdd(&short_rows, 1);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    status[0] = short_rows;
    status[1] = bad_rows;
  }
}

// What `move` does for pair i of a fork: row child[i] = the first whole[i] pages of row parent[i],
// then the fresh page dst[i] (none: -1), whose contents are those of page src[i]. whole -1: nothing.
struct ForkPlan {
  int32_t *whole, *src, *dst;
};

__global__ __launch_bounds__(kPlanThreads) void fork_plan_kernel(Books b, const int32_t* parents,
                                                                 const int32_t* children, int pairs,
                                                                 int32_t* status, ForkPlan plan,
                                                                 int32_t* list) {
  __shared__ int lds[kPlanWaves];
  __shared__ __attribute__((aligned(16))) int some_parents[kPlanThreads], some_children[kPlanThreads];
  __shared__ int taken[kPlanThreads];
  __shared__ int none_left, refused;
  if (threadIdx.x == 0) none_left = refused = 0;
  int want = 0;
  for (int base = 0; base < pairs; base += kPlanThreads) {
    const int i = base + (int)threadIdx.x;
    int need = 0, whole = -1;
    const int p = i < pairs ? parents[i] : -1, c = i < pairs ? children[i] : -1;
    // The child is no parent, and no earlier pair's child: four pairs to a read, the waves that hold
    // no pairs of their own taking parts of the others' (a plan of 64 pairs 6.5 us; with one read to a
    // pair, in every wave, 11.8).
    const int wave = (int)threadIdx.x >> 6, here = pairs - base < kPlanThreads ? pairs - base : kPlanThreads;
    const int waves = (here + 63) / 64, parts = kPlanWaves / waves, part = wave / waves;
    const int at = (wave - part * waves) * 64 + (int)(threadIdx.x & 63u);
    const int child = at < here ? children[base + at] : -1;
    bool found = false;
    taken[threadIdx.x] = 0;
    for (int from = 0; from < pairs; from += kPlanThreads) {
      const int mine = from + (int)threadIdx.x, n = pairs - from < kPlanThreads ? pairs - from : kPlanThreads;
      __syncthreads();
      some_parents[threadIdx.x] = mine < pairs ? parents[mine] : -1;  // (-1: no row's id)
      some_children[threadIdx.x] = mine < pairs ? children[mine] : -1;
      __syncthreads();
      const int share = ((n + 3) / 4 + parts - 1) / parts * 4, end = (part + 1) * share < n ? (part + 1) * share : n;
      if (part >= parts) continue;
#pragma unroll 4
      for (int k = part * share; k < end; k += 4) {
        const int4 x = *reinterpret_cast<const int4*>(some_parents + k);
        const int4 y = *reinterpret_cast<const int4*>(some_children + k);
        const int before = base + at - from - k;  // pairs of this read that come before the child's
        found |= x.x == child || x.y == child || x.z == child || x.w == child || (y.x == child && before > 0) ||
                 (y.y == child && before > 1) || (y.z == child && before > 2) || (y.w == child && before > 3);
      }
    }
    if (found) taken[at] = 1;
    __syncthreads();
    if (i < pairs) {
      const bool ok = p >= 0 && p < b.rows && c >= 0 && c < b.rows && !taken[threadIdx.x] && b.lens[c] == 0;
      if (ok) {
        const int len = clamp_len(b, b.lens[p]);
        whole = len / b.page;
        need = len % b.page != 0;
      } else {
        atomicAdd(&refused, 1);
      }
    }
    int total;
    const int rank = want + block_scan(need, lds, total);
    if (i < pairs) {
      plan.whole[i] = whole;
      plan.dst[i] = need ? rank : -1;
    }
    want += total;
  }
  const int found = rank_free(b, want, list, lds);
  __threadfence_block();
  __syncthreads();
  for (int i = threadIdx.x; i < pairs; i += kPlanThreads) {
    const int whole = plan.whole[i], rank = plan.dst[i];
    int src = -1, dst = -1;
    if (whole >= 0 && rank >= found) {
      atomicAdd(&none_left, 1);
      plan.whole[i] = -1;
    } else if (whole >= 0) {
      const int p = parents[i];
      if (rank >= 0) {
        dst = list[rank];
        src = b.table[(int64_t)p * b.width + whole];
        b.refs[dst] = 1;
      }
      b.lens[children[i]] = clamp_len(b, b.lens[p]);
    }
    plan.src[i] = src;
    plan.dst[i] = dst;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    status[0] = none_left;
    status[1] = refused;
  }
}

// Pages to move, from src[i] to dst[i], i < *count, and at[page] = i for each of them.
struct CompactPlan {
  int32_t *count, *src, *dst, *at;
};

__global__ __launch_bounds__(kPlanThreads) void compact_plan_kernel(Books b, int32_t* moved,
                                                                    CompactPlan plan) {
  __shared__ int lds[kPlanWaves];
  int live = 0;
  for (int base = 0; base < b.pages; base += kSlab) {
    int total;
    block_scan(__popc(held_bits(b.refs, b.pages, base)), lds, total);
    live += total;
  }
  int from = 0, to = 0;
  for (int base = 0; base < b.pages; base += kSlab) {
    const int first = base + (int)threadIdx.x * kSlabPer;
    const u32 held = held_bits(b.refs, b.pages, base), all = page_bits(b.pages, base);
    const int low = live - first;  // the thread's pages below `live`
    const u32 below = low <= 0 ? 0u : low >= kSlabPer ? (1u << kSlabPer) - 1u : (1u << low) - 1u;
    u32 out = held & ~below, in = ~held & all & below;
    int total;
    int rank = from + block_scan(__popc(out), lds, total);
    for (; out; out &= out - 1u) plan.src[rank++] = first + __ffs(out) - 1;
    from += total;
    rank = to + block_scan(__popc(in), lds, total);
    for (; in; in &= in - 1u) plan.dst[rank++] = first + __ffs(in) - 1;
    to += total;
  }
  // As many live pages lie above `live` as free ones below.
  __threadfence_block();
  __syncthreads();
  for (int i = threadIdx.x; i < from; i += kPlanThreads) {
    const int s = plan.src[i], d = plan.dst[i];
    plan.at[s] = i;
    b.refs[d] = b.refs[s];
    b.refs[s] = 0;
  }
  if (threadIdx.x == 0) {
    *plan.count = from;
    *moved = from;
  }
}

struct Pools {
  char* data[kMaxPools];
  int64_t bytes[kMaxPools];
};

enum Job : int { kCopy = 0, kFork = 1, kCompact = 2 };

// blockIdx.y < pools: pages of one pool, blockIdx.x over (move, part). blockIdx.y == pools: the
// table (fork: one pair a workgroup; compact: every live entry).
__global__ __launch_bounds__(kMoveThreads) void move_kernel(Pools pools, int n_pools, int job, Books b,
                                                            const int32_t* src, const int32_t* dst,
                                                            int count, const int32_t* device_count,
                                                            const int32_t* parents,
                                                            const int32_t* children,
                                                            const int32_t* whole,
                                                            const int32_t* index) {
  if ((int)blockIdx.y == n_pools) {
    if (job == kFork) {
      for (int i = blockIdx.x; i < count; i += gridDim.x) {
        if (whole[i] < 0) continue;
        const int32_t* from = b.table + (int64_t)parents[i] * b.width;
        int32_t* to = b.table + (int64_t)children[i] * b.width;
        for (int j = threadIdx.x; j < b.width; j += kMoveThreads) {
          int page = j == whole[i] ? dst[i] : -1;
          if (j < whole[i]) {
            page = from[j];
            if (page >= 0 && page < b.pages) atomicAdd(&b.refs[page], 1);
          }
          to[j] = page;
        }
      }
    } else {
      const int moves = *device_count;
      if (moves == 0) return;
      for (int r = blockIdx.x; r < b.rows; r += gridDim.x) {
        const int len = clamp_len(b, b.lens[r]), live = (int)(((int64_t)len + b.page - 1) / b.page);
        int32_t* row = b.table + (int64_t)r * b.width;
        for (int j = threadIdx.x; j < live; j += kMoveThreads) {
          const int page = row[j];
          if (page < 0 || page >= b.pages) continue;
          const int i = index[page];  // (written for pages that move, anything else otherwise)
          if (i >= 0 && i < moves && src[i] == page) row[j] = dst[i];
        }
      }
    }
    return;
  }
  const int64_t bytes = pools.bytes[blockIdx.y];
  char* const pool = pools.data[blockIdx.y];
  const int parts = (int)((bytes + kPart - 1) / kPart);
  const int moves = device_count ? *device_count : count;
  for (int64_t w = blockIdx.x; w < (int64_t)moves * parts; w += gridDim.x) {
    const int i = (int)(w / parts), part = (int)(w - (int64_t)i * parts);
    const int s = src[i], d = dst[i];
    if (s < 0 || s >= b.pages || d < 0 || d >= b.pages) continue;
    const char* from = pool + s * bytes + (int64_t)part * kPart;
    char* to = pool + d * bytes + (int64_t)part * kPart;
    const int64_t left = bytes - (int64_t)part * kPart;
    u32x4 x[kMoveLoads];
#pragma unroll
    for (int k = 0; k < kMoveLoads; ++k) {
      const int64_t at = (int64_t)(k * kMoveThreads + (int)threadIdx.x) * 16;
      if (at < left) x[k] = *reinterpret_cast<const u32x4*>(from + at);
    }
#pragma unroll
    for (int k = 0; k < kMoveLoads; ++k) {
      const int64_t at = (int64_t)(k * kMoveThreads + (int)threadIdx.x) * 16;
      if (at < left) __builtin_nontemporal_store(x[k], reinterpret_cast<u32x4*>(to + at));
    }
  }
}

// A live row holds its pages: given back by the first workgroup that takes its length.
__global__ __launch_bounds__(kMoveThreads) void free_kernel(Books b, const int32_t* rows) {
  __shared__ int taken;
  const int r = rows[blockIdx.x];
  if (r < 0 || r >= b.rows) return;
  if (threadIdx.x == 0) taken = atomicExch(&b.lens[r], 0);
  __syncthreads();
  const int len = clamp_len(b, taken);
  if (len == 0) return;
  const int live = (int)(((int64_t)len + b.page - 1) / b.page);
  int32_t* row = b.table + (int64_t)r * b.width;
  for (int j = threadIdx.x; j < b.width; j += kMoveThreads) {
    const int page = row[j];
    if (j < live && page >= 0 && page < b.pages) atomicSub(&b.refs[page], 1);
    row[j] = -1;
  }
}

static int check_pools(const fgw_pages_pools* p) {
  if (!p || p->count < 0 || (p->count > 0 && (!p->data || !p->page_bytes)))
    return fail(FGW_MHA_EINVAL, "pools are missing");
  for (int i = 0; i < p->count; ++i)
    if (!p->data[i] || !aligned16(p->data[i]) || p->page_bytes[i] <= 0 || p->page_bytes[i] % 16)
      return fail(FGW_MHA_EINVAL, "pools must be 16-byte aligned, their pages multiples of 16 bytes");
  return FGW_MHA_OK;
}

// The pools in launches of kMaxPools, the table with the first. Workgroups of a pool: its moves'
// parts; where only the device knows how many moves there are, kMovers over all pools of the launch
// and at least 64 a pool, which walk them in a loop (205 moves, us, 2048 / 4096 / 8192: 50 / 48 / 45; with
// nothing to move the call takes no longer).
static int launch_moves(const fgw_pages_pools* pools, Job job, const Books& b, const int32_t* src,
                        const int32_t* dst, int count, const int32_t* device_count,
                        const int32_t* parents, const int32_t* children, const int32_t* whole,
                        const int32_t* index, hipStream_t stream) {
  int done = 0;
  do {
    Pools arg = {};
    const int n = std::min(kMaxPools, pools->count - done);
    int64_t parts = 1;
    for (int i = 0; i < n; ++i) {
      arg.data[i] = static_cast<char*>(pools->data[done + i]);
      arg.bytes[i] = pools->page_bytes[done + i];
      parts = std::max(parts, (arg.bytes[i] + kPart - 1) / kPart);
    }
    const bool table = done == 0 && job != kCopy;
    const int64_t wanted = std::max<int64_t>(1, (int64_t)count * parts);
    const int64_t most = device_count ? std::max(64, kMovers / std::max(1, n)) : 1 << 20;
    const unsigned x = (unsigned)std::min(wanted, most), y = (unsigned)(n + (table ? 1 : 0));
    if (y == 0) break;
    move_kernel<<<dim3(x, y), dim3(kMoveThreads), 0, stream>>>(arg, n, job, b, src, dst, count,
                                                               device_count, parents, children,
                                                               whole, index);
    if (int rc = launched("fgw_pages")) return rc;
    done += n;
  } while (done < pools->count);
  return FGW_MHA_OK;
}

}  // namespace fgw_kv

using namespace fgw_kv;

extern "C" {

// reserve: entries + 1 sums and a list of the pages; fork: whole, src, dst and a list; compact:
// the number of moves, src, dst and each page's place among them.
int64_t fgw_pages_workspace(int32_t pages, int32_t entries) {
  return 4 * ((int64_t)std::max(entries, 0) + 1) + 2 * ((int64_t)std::max(pages, 0) + 4);
}

int fgw_pages_reserve(const fgw_pages_books* books, const int32_t* counts, int32_t* status,
                      int32_t* workspace, hipStream_t stream) {
  Books b;
  if (int rc = check_books(books, b)) return rc;
  if (!counts || !status || !workspace) return fail(FGW_MHA_EINVAL, "tensors are missing");
  reserve_kernel<<<dim3(1), dim3(kPlanThreads), 0, stream>>>(b, counts, status, workspace);
  return launched("fgw_pages_reserve");
}

int fgw_pages_fork(const fgw_pages_books* books, const fgw_pages_pools* pools,
                   const int32_t* parents, const int32_t* children, int32_t pairs, int32_t* status,
                   int32_t* workspace, hipStream_t stream) {
  Books b;
  if (int rc = check_books(books, b)) return rc;
  if (int rc = check_pools(pools)) return rc;
  if (pairs < 0 || !status || !workspace || (pairs > 0 && (!parents || !children)))
    return fail(FGW_MHA_EINVAL, "tensors are missing");
  const ForkPlan plan{workspace, workspace + pairs, workspace + 2 * (int64_t)pairs};
  fork_plan_kernel<<<dim3(1), dim3(kPlanThreads), 0, stream>>>(b, parents, children, pairs, status,
                                                               plan, workspace + 3 * (int64_t)pairs);
  if (int rc = launched("fgw_pages_fork")) return rc;
  if (pairs == 0) return FGW_MHA_OK;
  return launch_moves(pools, kFork, b, plan.src, plan.dst, pairs, nullptr, parents, children,
                      plan.whole, nullptr, stream);
}

int fgw_pages_free(const fgw_pages_books* books, const int32_t* rows, int32_t count,
                   hipStream_t stream) {
  Books b;
  if (int rc = check_books(books, b)) return rc;
  if (count < 0 || (count > 0 && !rows)) return fail(FGW_MHA_EINVAL, "tensors are missing");
  if (count == 0) return FGW_MHA_OK;
  free_kernel<<<dim3((unsigned)count), dim3(kMoveThreads), 0, stream>>>(b, rows);
  return launched("fgw_pages_free");
}

int fgw_pages_compact(const fgw_pages_books* books, const fgw_pages_pools* pools, int32_t* moved,
                      int32_t* workspace, hipStream_t stream) {
  Books b;
  if (int rc = check_books(books, b)) return rc;
  if (int rc = check_pools(pools)) return rc;
  if (!moved || !workspace) return fail(FGW_MHA_EINVAL, "tensors are missing");
  const int64_t half = b.pages / 2 + 1;  // no more pages move than half of them
  const CompactPlan plan{workspace, workspace + 1, workspace + 1 + half, workspace + 1 + 2 * half};
  compact_plan_kernel<<<dim3(1), dim3(kPlanThreads), 0, stream>>>(b, moved, plan);
  if (int rc = launched("fgw_pages_compact")) return rc;
  return launch_moves(pools, kCompact, b, plan.src, plan.dst,
                      (int)std::max<int64_t>(half - 1, b.rows), plan.count, nullptr, nullptr,
                      nullptr, plan.at, stream);
}

int fgw_pages_copy(const fgw_pages_pools* pools, int32_t pages, const int32_t* src,
                   const int32_t* dst, int32_t count, hipStream_t stream) {
  if (int rc = check_pools(pools)) return rc;
  if (pages <= 0 || count < 0 || (count > 0 && (!src || !dst)))
    return fail(FGW_MHA_EINVAL, "tensors are missing");
  if (count == 0) return FGW_MHA_OK;
  Books b = {};
  b.pages = pages;
  return launch_moves(pools, kCopy, b, src, dst, count, nullptr, nullptr, nullptr, nullptr, nullptr,
                      stream);
}

}  // extern "C"
