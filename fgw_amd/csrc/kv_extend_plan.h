// Host side of the attention over pages with grouped heads, for the entry points that launch its kernels
// (kv_extend.hip, kv_shared.hip): which kernel takes which requests, grids, workspace, checks.
#pragma once
#include <algorithm>

#include "kv_common.h"
#include "kv_extend.h"
#include "kv_extend_long.h"
#include "kv_extend_wide.h"

namespace fgw_kv {

// Requests of up to kLongFrom rows (tokens times query heads of a K/V head) take the kernel of few
// rows: it reads the keys once for every 32 of them, the long one once for 256. Hq 32, Hkv 8, D 128,
// pages of 64, few rows / long, us: 128 rows B1 KV 1024 17.7 / 17.6, B4 KV 2048 27.6 / 30.6, B1 KV
// 8192 29.3 / 27.0, B8 KV 8192 112 / 88; 192 rows 18.3 / 19.6, 34.0 / 32.3, 36.2 / 29.4, 184 / 92.
constexpr int kLongFrom = 128;
// Units of a split at least (rounds of 128 keys, blocks of 64): below, a split's own cost outweighs
// what it saves. Few rows, B1 Hq 32 Hkv 8 D 128, splits of 1 / 2 / 4 rounds, us: KV 1024
// 10.5 / 11.3 / 14.3, 2048 10.8 / 12.1 / 14.6; long, B1 100 tokens KV 1000, 4 / 8 blocks: 26.1 / 32.4.
constexpr int kRowsMinChunk = 1, kLongMinChunk = 4;
// Rounds of a tile of few rows that is never split: one takes 0.9 us at D 64, 1.35 at D 128, the join
// 3 us. Whole / split, us: D 64 KV 384 7.6 / 9.2, 512 8.6 / 9.0, 768 10.4 / 9.4; D 128 KV 384 9.6 / 10.2,
// 512 11.0 / 10.0.
constexpr int kRowsWhole = 3, kRowsWholeNarrow = 4;  // (D <= 64)
// Rounds of a tile above which a split has two: a join takes 0.14 us for every split of 4 rows, 0.3 of
// 16. Splits of 1 / 2, us: 4 rows (the case above) 16 rounds 10.8 / 12.1, 32 rounds 13.9 / 13.1; 16 rows
// (Hkv 2) 8 rounds 12.4 / 13.4, 16 rounds 14.8 / 13.9.
constexpr int kRowsMany = 16, kRowsManyTall = 8;  // (requests of more than 8 rows)

// Compute units that a call fills at most: those of the card. They bound splits and workspace (256
// places of 132 KB), so that offsets of partials that a launch joins itself and the products of split_bound
// stay in 32 bits whatever num_cus a caller gives.
constexpr int kMostCus = 256;
static_assert(kMostCus <= fgw_mha::kMostSplits, "split_bound");

template <class P>
using ExtendLaunch = hipError_t (*)(const P&, int, hipStream_t);

template <bool BF16, class P>
inline ExtendLaunch<P> rows_entry(int dim) {
  return dim <= 32    ? &launch_extend_rows<BF16, 32, P>
         : dim <= 64  ? &launch_extend_rows<BF16, 64, P>
         : dim <= 128 ? &launch_extend_rows<BF16, 128, P>
                      : &launch_extend_rows<BF16, 256, P>;
}

// Keys of one DMA instruction: 1024 bytes / (2 * head-dim tile).
template <bool BF16, class P>
inline ExtendLaunch<P> long_entry(int dim, int page) {
  if (dim > 128) return &launch_extend_wide<BF16, 256, P>;
  if (dim == 128)
    return page % LongTiling::BN == 0 ? &launch_extend_long<BF16, 128, kRowsBlock, P>
           : page % 4 == 0        ? &launch_extend_long<BF16, 128, kRowsGroup, P>
                                  : &launch_extend_long<BF16, 128, kRowsPadded, P>;
  if (dim == 64)
    return page % LongTiling::BN == 0 ? &launch_extend_long<BF16, 64, kRowsBlock, P>
           : page % 8 == 0        ? &launch_extend_long<BF16, 64, kRowsGroup, P>
                                  : &launch_extend_long<BF16, 64, kRowsPadded, P>;
  return dim < 64 ? &launch_extend_long<BF16, 64, kRowsPadded, P> : &launch_extend_long<BF16, 128, kRowsPadded, P>;
}

// One launch of a kernel over the requests with rows_from < n * group <= rows_to.
struct Launch {
  int rows_from, rows_to;
  int target, min_chunk, whole, many;  // ExtendParams
  int64_t tiles;             // at most, of one K/V head
  int64_t items;             // at most: the grid; 0: no launch
  int64_t slots;             // places for partials and notes
  int64_t floats, counters;  // of workspace
};

// Splits of a tile at most: of the table's capacity, or the window's span (which begins anywhere in a
// unit).
template <class T>
inline int64_t most_splits(const fgw_kv_extend_args& a, int min_chunk, int whole) {
  int64_t keys = (int64_t)a.width * a.page_size;
  if (a.window > 0) keys = std::min<int64_t>(keys, (int64_t)a.window + a.max_new);
  const int64_t units = (keys + T::KEYS - 1) / T::KEYS + (a.window > 0);
  return units <= whole ? 1 : (units + min_chunk - 1) / min_chunk;
}

// Grid and workspace of a launch: where tiles may be split (best_chunk) all items together are at
// most one to a CU; else there are as many as tiles.
template <class T>
inline void plan_items(Launch& l, const fgw_kv_extend_args& a, bool may_split) {
  l.items = l.tiles * a.kv_heads;
  const int64_t most = most_splits<T>(a, l.min_chunk, l.whole);
  if (!may_split || most <= 1 || a.num_cus / a.kv_heads <= 1) return;
  l.target = a.num_cus;
  l.slots = std::min<int64_t>(l.target, l.items * most);
  l.items = std::max(l.items, l.slots);
  l.floats = l.slots * (T::ROWS * (a.dim + 1) + (int64_t)sizeof(JoinNote) / 4);
}

struct Plan {
  Launch rows, longs;
};

inline Plan plan(fgw_kv_extend_args a) {
  a.num_cus = std::min(a.num_cus, kMostCus);
  const int64_t group = a.heads / a.kv_heads, total = a.tokens * group;
  const int64_t rows_most = std::min(a.max_new, a.tokens) * group, batch = std::min(a.batch, a.tokens);
  auto tiles = [&](int64_t requests, int64_t rows, int64_t tile) {  // of so many requests at most
    return std::min(requests * ((rows + tile - 1) / tile), total / tile + requests);
  };
  Plan p = {};
  // (One request is as long as the sizes say, unless q has rows behind it: no second launch for a short
  // one. Two launches / one, us: 100 tokens of 1000 25.7 / 23.2, 512 of 8192 87.4 / 83.6.)
  const bool only_long = a.batch == 1 && rows_most > kLongFrom;
  if (!only_long) {
    p.rows.rows_to = kLongFrom;
    p.rows.min_chunk = kRowsMinChunk;
    p.rows.whole = a.dim <= 64 ? kRowsWholeNarrow : kRowsWhole;
    p.rows.many = rows_most <= 8 ? kRowsMany : kRowsManyTall;
    p.rows.tiles = tiles(batch, std::min<int64_t>(rows_most, kLongFrom), ShortTiling::ROWS);
    plan_items<ShortTiling>(p.rows, a, true);
    p.rows.counters = p.rows.slots * fgw_mha::kArrivalStride;
  }
  if (rows_most > kLongFrom) {
    p.longs.rows_from = only_long ? 0 : kLongFrom;
    p.longs.rows_to = 0x7fffffff;
    p.longs.min_chunk = kLongMinChunk;
    p.longs.many = 1 << 20;
    // (So many tokens that whole tiles fill the card four times over, unless most of them are
    // padding: no workspace, and no launch for joins.)
    const int64_t requests = std::min(batch, only_long ? 1 : total / kLongFrom);
    auto longs = [&](auto tiling) {
      using T = decltype(tiling);
      p.longs.tiles = tiles(requests, rows_most, T::ROWS);
      plan_items<T>(p.longs, a, total / T::ROWS * a.kv_heads < 4 * (int64_t)a.num_cus);
    };
    if (a.dim > 128) longs(WideTiling{}); else longs(LongTiling{});
  }
  return p;
}

inline int check(const fgw_kv_extend_args* a) {
  if (!a) return fail(FGW_MHA_EINVAL, "arguments are missing");
  if (a->dtype != FGW_KV_FLOAT16 && a->dtype != FGW_KV_BFLOAT16)
    return fail(FGW_MHA_EUNSUPPORTED, "matching FP16/BF16 Q/K/V required");
  if (a->dim < 16 || a->dim > 256 || a->dim % 16)
    return fail(FGW_MHA_EUNSUPPORTED, "D must be in [16, 256] and divisible by 16");
  if (a->page_size <= 0 || a->pool_rows <= 0 || a->pool_rows % a->page_size || a->width <= 0)
    return fail(FGW_MHA_EINVAL,
                "positive page size, whole pool pages and positive table width required");
  if ((int64_t)a->width * a->page_size > 0x7fffffff - 0x10000)
    return fail(FGW_MHA_EUNSUPPORTED, "table capacity must fit in 31 bits");
  if (a->tokens < 0 || a->batch <= 0 || a->heads <= 0 || a->kv_heads <= 0 || a->max_new <= 0 ||
      a->num_cus <= 0)
    return fail(FGW_MHA_EINVAL, "positive extents required");
  if (a->heads % a->kv_heads)
    return fail(FGW_MHA_EINVAL, "query heads must be a multiple of the K/V heads");
  if (a->window < 0 || (a->window > 0 && !a->causal))
    return fail(FGW_MHA_EINVAL, "a window must be positive and needs causal attention");
  if (!(a->scale > 0.0f) || a->scale > 3.0e38f)
    return fail(FGW_MHA_EINVAL, "the scale of the scores must be positive and finite");
  if ((int64_t)a->tokens * (a->heads / a->kv_heads) > 0x7fffffff - 0x10000)
    return fail(FGW_MHA_EUNSUPPORTED, "too many rows for one call");
  return FGW_MHA_OK;
}

// The launches of a plan over the workspace base.parts.
template <bool BF16, class P>
inline int run(const P& base, const Plan& plan, const char* name, hipStream_t stream) {
  P rows = base, longs = base;
  float* work = base.parts;
  auto place = [&](P& p, const Launch& l, int rows_tile) {
    p.rows_from = l.rows_from;
    p.rows_to = l.rows_to;
    p.target = l.target;
    p.min_chunk = l.min_chunk;
    p.whole = l.whole;
    p.many = l.many;
    p.work = (int)l.slots;
    p.notes = l.target > 0 && !p.counters ? reinterpret_cast<int32_t*>(work + l.slots * rows_tile * (p.dim + 1)) : nullptr;
    p.parts = work;
    p.lse = work + l.slots * rows_tile * p.dim;
    work += l.floats;
  };
  longs.counters = nullptr;
  place(rows, plan.rows, ShortTiling::ROWS);
  place(longs, plan.longs, base.dim > 128 ? WideTiling::ROWS : LongTiling::ROWS);
  hipError_t e = hipSuccess;
  if (plan.longs.items > 0) e = long_entry<BF16, P>(base.dim, base.page_size)(longs, (int)plan.longs.items, stream);
  if (e == hipSuccess && plan.rows.items > 0) e = rows_entry<BF16, P>(base.dim)(rows, (int)plan.rows.items, stream);
  if (e != hipSuccess) return fail(FGW_MHA_EHIP, "%s: %s", name, hipGetErrorString(e));
  const int rows_items = rows.notes ? rows.work : 0, long_items = longs.notes ? longs.work : 0;
  if (rows_items + long_items == 0) return FGW_MHA_OK;
  extend_join_kernel<BF16, P><<<dim3((unsigned)(rows_items + long_items), long_items > 0 ? kJoinParts : 1),
                             dim3(kMergeThreads), 0, stream>>>(rows, longs, rows_items);
  return launched(name);
}

inline int check_tensors(const fgw_kv_extend_args& a) {
  if (!a.q.data || !a.out || !a.k_cache || !a.v_cache || !a.block_table || !a.cache_seqlens || !a.cu_seqlens)
    return fail(FGW_MHA_EINVAL, "tensors are missing");
  if (!aligned16(a.q.data) || !aligned16(a.out) || !aligned16(a.k_cache) || !aligned16(a.v_cache) ||
      a.q.token_stride % 8 || a.q.head_stride % 8)
    return fail(FGW_MHA_EINVAL, "rows must be 16-byte aligned, their strides multiples of 16 bytes");
  return FGW_MHA_OK;
}

// The fields of P that follow from the arguments alone.
template <class P>
inline P params_of(const fgw_kv_extend_args& a) {
  P p = {};
  p.q = a.q.data;
  p.q_token = a.q.token_stride * 2;
  p.q_head = a.q.head_stride * 2;
  p.k = a.k_cache;
  p.v = a.v_cache;
  p.table = a.block_table;
  p.lengths = a.cache_seqlens;
  p.cu = a.cu_seqlens;
  p.out = a.out;
  p.pool_rows = a.pool_rows;
  p.batch = a.batch;
  p.heads = a.kv_heads;
  p.dim = a.dim;
  p.width = a.width;
  p.page_size = a.page_size;
  p.causal = a.causal != 0;
  page_division((uint32_t)a.page_size, p.page_magic, p.page_shift);
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.tokens = a.tokens;
  p.q_heads = a.heads;
  p.group = a.heads / a.kv_heads;
  p.max_new = std::min(a.max_new, a.tokens);
  // (No key lies as far back as the table's capacity.)
  p.window = a.window < (int64_t)a.width * a.page_size ? a.window : 0;
  return p;
}

}  // namespace fgw_kv
