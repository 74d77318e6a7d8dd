// C ABI of the attention weight of cached keys (fgw_kv_weights): checks, sizes and dispatch. The kernels
// stand in kv_weights.h, their instantiations in the kv_weights_*.hip files of each type.
#include <hip/hip_runtime.h>

#include "kv_extend_plan.h"
#include "kv_weights.h"

namespace fgw_kv {

#define FGW_KV_EXTERN_WEIGHTS(BF, DP)                                                              \
  extern template hipError_t launch_weights<BF, DP>(const WeightParams&, bool, int, hipStream_t); \
  extern template hipError_t launch_weights_columns<BF, DP>(const WeightParams&, int, hipStream_t);
FGW_KV_EXTERN_WEIGHTS(true, 64) FGW_KV_EXTERN_WEIGHTS(true, 128) FGW_KV_EXTERN_WEIGHTS(true, 256)
FGW_KV_EXTERN_WEIGHTS(false, 64) FGW_KV_EXTERN_WEIGHTS(false, 128) FGW_KV_EXTERN_WEIGHTS(false, 256)

namespace {

// Items of weights_stats_kernel, two to a CU, where its tiles are fewer. 256 / 512 / 1024 items, us of a call:
// 2000 tokens of 2 K/V heads of 8 rows 75.0 / 74.3 / 81.0, 64 requests of 17 tokens 92.9 / 93.0 / 97.8.
constexpr int kStatsItems = 512;

// Items of weights_rows_kernel: two to a CU, and the three that it holds where the requests alone fill the card,
// so that ragged ones even out. 512 / 768 / 1024 items, us: 32 requests of 8 K/V heads, 1 to 8192 keys 92.8 /
// 86.0 / 93.0, all of 8192 keys 124.6 / 125.0 / 131.8, 64 of 2048 63.8 / 66.0 / 72.6; 8 of 8192, of few
// requests, 37.8 at 512 and 42.5 at 1024 (256: 40.3).
constexpr int kFewItems = 512, kManyItems = 768;
static_assert(std::max({kStatsItems, kFewItems, kManyItems}) <= fgw_mha::kMostSplits, "split_bound");

// Bytes of kept scores, or of partial sums, that a call may always ask for; else as many as the pool has.
constexpr int64_t kKeptBytes = 256 << 20;

struct WeightPlan {
  bool many;       // rows of a request and K/V head, at most, past kKeptRows, or too many scores to keep
  Launch launch;   // of the first pass
  int part_rows;
  int columns, sums;  // grids of the persistent kernels; 0: no launch
  int blocks, step;   // of kColumnKeys keys: of the table, of one launch of those kernels
  int64_t keys_pad, kept_rows, parts;
  int64_t kept, lse, notes, floats;  // of workspace
};

// Workgroups of a persistent kernel: as many as the card holds, or as there are items.
int persistent(int64_t items, int num_cus, int each) { return (int)std::min<int64_t>(items, (int64_t)num_cus * each); }

// The extents that plan_items reads.
fgw_kv_extend_args extents(const fgw_kv_weights_args& a) {
  fgw_kv_extend_args e = {};
  e.tokens = a.tokens;
  e.batch = a.batch;
  e.heads = a.heads;
  e.kv_heads = a.kv_heads;
  e.dim = a.dim;
  e.width = a.width;
  e.page_size = a.page_size;
  e.pool_rows = a.pool_rows;
  e.max_new = a.last;
  e.causal = 1;
  e.dtype = a.dtype;
  e.num_cus = std::min(a.num_cus, kMostCus);
  e.scale = a.scale;
  e.q = a.q;
  e.k_cache = a.k_cache;
  e.block_table = a.block_table;
  e.cache_seqlens = a.cache_seqlens;
  e.cu_seqlens = a.cu_seqlens;
  return e;
}

WeightPlan plan_weights(const fgw_kv_weights_args& a) {
  const fgw_kv_extend_args e = extents(a);
  WeightPlan p = {};
  const int64_t group = a.heads / a.kv_heads, total = a.tokens * group, capacity = (int64_t)a.width * a.page_size;
  const int64_t rows = std::min(a.last, a.tokens) * group, requests = std::min(a.batch, a.tokens);
  auto blocks = [&](int64_t size) { return std::min(requests * ((rows + size - 1) / size), total / size + requests); };
  p.blocks = p.step = (int)((capacity + kColumnKeys - 1) / kColumnKeys);
  p.keys_pad = (int64_t)p.blocks * kColumnKeys;
  // (Kept scores have a place for every key that the table could hold: no more of them than the pool has bytes.)
  const int64_t kept = (int64_t)a.batch * a.kv_heads * rows * p.keys_pad;
  const int64_t bound = std::max<int64_t>(kKeptBytes, a.pool_rows * a.kv_heads * a.dim * 2);
  p.many = rows > (a.dim <= 128 ? kKeptRows : kKeptRowsWide) || kept * 4 > bound;
  if (!p.many) {
    p.launch.min_chunk = kRowsMinChunk;
    p.launch.whole = a.dim <= 64 ? kRowsWholeNarrow : kRowsWhole;
    p.launch.many = rows <= 8 ? kRowsMany : kRowsManyTall;
    p.launch.tiles = requests;
    fgw_kv_extend_args rounds = e;
    rounds.num_cus = p.launch.tiles * a.kv_heads >= e.num_cus ? kManyItems : kFewItems;
    plan_items<KeptTiling<1>>(p.launch, rounds, true);  // (the same for tiles of 64 rows)
    p.kept_rows = rows;
    p.kept = kept;
    p.lse = p.launch.slots * (rows <= 32 ? 32 : 64);
  } else {
    p.launch.min_chunk = kLongMinChunk;
    p.launch.many = 1 << 20;
    p.launch.tiles = blocks(StatsTiling::ROWS);
    p.launch.items = p.launch.tiles * a.kv_heads;
    // (Statistics of a split are a number a row: as many splits as even out the causal tiles.)
    const int64_t most = most_splits<StatsTiling>(e, p.launch.min_chunk, 0);
    if (most > 1) {
      p.launch.target = kStatsItems;
      p.launch.items = std::max(p.launch.items, std::min<int64_t>(p.launch.target, p.launch.items * most));
    }
    p.launch.slots = p.launch.items;  // every item leaves statistics
    p.lse = p.launch.slots * StatsTiling::ROWS;
    p.notes = (int64_t)a.batch * (int64_t)sizeof(WeightNote) / 4;
    // Parts of the rows: smaller ones where the items would not fill the card (half of them: causal), down to
    // what a program of its own is worth. Parts of 1024 rows always / by this rule, us of a call: 512 tokens of
    // one K/V head of 8 rows 55.5 / 35.9, 4 requests of 300 tokens 53.4 / 35.8, 2000 tokens of 2 heads 77.4 / 74.3.
    p.part_rows = kColumnRows;
    while (p.part_rows > kColumnRows / 4 && rows > p.part_rows / 2 &&
           total / p.part_rows * p.blocks * a.kv_heads < 4 * (int64_t)e.num_cus)
      p.part_rows /= 2;
    if (rows > p.part_rows) {
      // Places for the sums of every part (of requests with several) and key, by the table's capacity: where those
      // are too many, the keys are taken a range at a time, with the same sums.
      p.parts = std::min(requests * ((rows + p.part_rows - 1) / p.part_rows),
                         total / p.part_rows + std::min(requests, total / p.part_rows));
      const int64_t block = p.parts * a.kv_heads * kColumnKeys;
      p.step = (int)std::max<int64_t>(1, std::min<int64_t>(p.blocks, bound / (4 * block)));
      p.keys_pad = (int64_t)p.step * kColumnKeys;
      p.kept = p.step * block;
      p.sums = persistent(requests * p.step * a.kv_heads, e.num_cus, 4);
    }
    p.columns = persistent(blocks(p.part_rows) * p.step * a.kv_heads, e.num_cus, a.dim > 128 ? 1 : 2);
  }
  p.floats = p.kept + (p.lse + 3) / 4 * 4 + p.notes;
  return p;
}

int check_weights(const fgw_kv_weights_args* args) {
  if (!args) return fail(FGW_MHA_EINVAL, "arguments are missing");
  if (args->last <= 0) return fail(FGW_MHA_EINVAL, "the number of tokens that count must be positive");
  const fgw_kv_extend_args e = extents(*args);
  if (int rc = check(&e)) return rc;
  if (!(args->decay >= 0.0f) || args->decay > 3.0e38f)
    return fail(FGW_MHA_EINVAL, "the decay must be finite and not negative");
  if (args->scores_stride < (int64_t)args->width * args->page_size)
    return fail(FGW_MHA_EINVAL, "the scores must have a place for every key of the table");
  const int64_t rows = (int64_t)args->tokens * (args->heads / args->kv_heads);
  const int64_t keys = (int64_t)args->width * args->page_size / kColumnKeys + 1;
  if ((rows / (kColumnRows / 4) + args->batch) * keys > 0x3fffffff)
    return fail(FGW_MHA_EUNSUPPORTED, "too many rows for one call");
  return FGW_MHA_OK;
}

template <bool BF16>
hipError_t launch(const WeightParams& w, const WeightPlan& p, hipStream_t stream) {
  return w.dim <= 64    ? launch_weights<BF16, 64>(w, p.many, (int)p.launch.items, stream)
         : w.dim <= 128 ? launch_weights<BF16, 128>(w, p.many, (int)p.launch.items, stream)
                        : launch_weights<BF16, 256>(w, p.many, (int)p.launch.items, stream);
}
template <bool BF16>
hipError_t launch_columns(const WeightParams& w, const WeightPlan& p, hipStream_t stream) {
  return w.dim <= 64    ? launch_weights_columns<BF16, 64>(w, p.columns, stream)
         : w.dim <= 128 ? launch_weights_columns<BF16, 128>(w, p.columns, stream)
                        : launch_weights_columns<BF16, 256>(w, p.columns, stream);
}

}  // namespace

}  // namespace fgw_kv

using namespace fgw_kv;

extern "C" {

int64_t fgw_kv_weights_workspace(const fgw_kv_weights_args* args) {
  if (int rc = check_weights(args)) return rc;
  return args->tokens == 0 ? 0 : plan_weights(*args).floats;
}

int fgw_kv_weights(const fgw_kv_weights_args* args, hipStream_t stream) {
  if (int rc = check_weights(args)) return rc;
  const fgw_kv_weights_args& a = *args;
  if (a.tokens == 0) return FGW_MHA_OK;
  if (!a.q.data || !a.scores || !a.k_cache || !a.block_table || !a.cache_seqlens || !a.cu_seqlens)
    return fail(FGW_MHA_EINVAL, "tensors are missing");
  if (!aligned16(a.q.data) || !aligned16(a.k_cache) || a.q.token_stride % 8 || a.q.head_stride % 8)
    return fail(FGW_MHA_EINVAL, "rows must be 16-byte aligned, their strides multiples of 16 bytes");
  const WeightPlan p = plan_weights(a);
  if (p.launch.items > 0x3fffffff) return fail(FGW_MHA_EUNSUPPORTED, "too many rows for one call");
  if (p.floats > 0 && (!a.workspace || !aligned16(a.workspace))) return fail(FGW_MHA_EINVAL, "the workspace is missing");
  WeightParams w = params_of<WeightParams>(extents(a));
  w.max_new = w.tokens;
  w.scores = a.scores;
  w.stride = a.scores_stride;
  w.last = a.last;
  w.decay = a.decay;
  w.part_rows = p.part_rows;
  for (w.part_shift = 0; w.part_rows > 1 << w.part_shift;) ++w.part_shift;
  w.keys_pad = (int32_t)p.keys_pad;
  w.kept_rows = (int32_t)p.kept_rows;
  w.parts_most = (int32_t)p.parts;
  w.target = p.launch.target;
  w.min_chunk = p.launch.min_chunk;
  w.whole = p.launch.whole;
  w.many = p.launch.many;
  w.work = (int32_t)p.launch.slots;
  w.kept = w.sums = a.workspace;
  w.lse = a.workspace + p.kept;
  w.request_notes = reinterpret_cast<int32_t*>(w.lse + (p.lse + 3) / 4 * 4);
  const hipError_t e = a.dtype == FGW_KV_BFLOAT16 ? launch<true>(w, p, stream) : launch<false>(w, p, stream);
  if (e != hipSuccess) return fail(FGW_MHA_EHIP, "fgw_kv_weights: %s", hipGetErrorString(e));
  if (!p.many && p.launch.target > 0) {
    if (w.kept_rows <= 32)
      weights_finish_kernel<1><<<dim3((unsigned)p.launch.items), dim3(kFinishThreads), 0, stream>>>(w, w.lengths, w.cu);
    else
      weights_finish_kernel<2><<<dim3((unsigned)p.launch.items), dim3(kFinishThreads), 0, stream>>>(w, w.lengths, w.cu);
  }
  for (int from = 0; p.many && from < p.blocks; from += p.step) {
    w.block_from = from;
    w.block_to = std::min(from + p.step, p.blocks);
    const hipError_t c = a.dtype == FGW_KV_BFLOAT16 ? launch_columns<true>(w, p, stream) : launch_columns<false>(w, p, stream);
    if (c != hipSuccess) return fail(FGW_MHA_EHIP, "fgw_kv_weights: %s", hipGetErrorString(c));
    if (p.sums > 0)
      weights_sum_kernel<<<dim3((unsigned)p.sums), dim3(kFinishThreads), 0, stream>>>(w, w.lengths, w.cu);
  }
  return launched("fgw_kv_weights");
}

}  // extern "C"
