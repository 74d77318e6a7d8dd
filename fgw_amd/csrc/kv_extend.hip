// C ABI of the attention over pages with grouped heads: checks, sizes and dispatch. The kernels
// stand in kv_extend.h, their instantiations in kv_extend_bf16.hip and kv_extend_f16.hip.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kv_common.h"
#include "kv_extend.h"

namespace fgw_kv {

#define FGW_KV_EXTERN_ROWS(BF, DP) \
  extern template hipError_t launch_extend_rows<BF, DP>(const ExtendParams&, int, hipStream_t);
FGW_KV_EXTERN_ROWS(true, 32) FGW_KV_EXTERN_ROWS(true, 64)
FGW_KV_EXTERN_ROWS(true, 128) FGW_KV_EXTERN_ROWS(true, 256)
FGW_KV_EXTERN_ROWS(false, 32) FGW_KV_EXTERN_ROWS(false, 64)
FGW_KV_EXTERN_ROWS(false, 128) FGW_KV_EXTERN_ROWS(false, 256)

namespace {

constexpr int kRowsTile = 32, kRowsBlock = 32;

int dim_tile(int dim) { return dim <= 32 ? 32 : dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// One launch of a kernel: its items at most, and whether tiles may be split.
struct Launch {
  int64_t tiles;  // at most, of one K/V head
  int64_t items;  // at most: the grid
  int target, min_chunk;
  int64_t floats;  // of workspace
  int rows_tile;
};

// find_item cuts a tile into at most blocks / chunk + 1 splits with chunk >= visits / target, so
// there are at most target + tiles * kv_heads items (and two for the rounding of the sum), and no
// more than every tile cut as far as the table's capacity allows.
Launch plan_launch(const fgw_kv_extend_args& a, int64_t tiles, int64_t tiles_sure, int rows_tile,
                   int block, int target, int min_chunk) {
  const int64_t capacity = (int64_t)a.width * a.page_size;
  int64_t keys = capacity;
  if (a.window > 0) keys = std::min<int64_t>(keys, (int64_t)a.window + a.max_new);
  const int64_t blocks = (keys + block - 1) / block + 1;
  const int64_t most = (blocks + min_chunk - 1) / min_chunk;
  Launch l{tiles, tiles * a.kv_heads, 0, min_chunk, 0, rows_tile};
  if (most > 1 && tiles_sure * a.kv_heads < 4 * (int64_t)target) {
    l.target = target;
    l.items = std::min(tiles * a.kv_heads * most, target + target / 1024 + 2 + tiles * a.kv_heads);
    l.floats = l.items * rows_tile * (a.dim + 1);
  }
  return l;
}

Launch plan_rows(const fgw_kv_extend_args& a) {
  const int64_t group = a.heads / a.kv_heads;
  const int64_t most = std::min<int64_t>(a.max_new, a.tokens);
  const int64_t tiles = std::min<int64_t>(a.batch * ((most * group + kRowsTile - 1) / kRowsTile),
                                          a.tokens * group / kRowsTile + std::min(a.batch, a.tokens));
  const int64_t sure = std::max<int64_t>(a.tokens * group / kRowsTile, a.tokens / most);
  return plan_launch(a, tiles, sure, kRowsTile, kRowsBlock, 2 * a.num_cus, 8);
}

int check(const fgw_kv_extend_args* a) {
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

}  // namespace

// At most `tiles` tiles of a launch; joins take 16 rows' workgroups of a tile each.
template <bool BF16>
static int run_rows(const ExtendParams& p, const Launch& l, int dpad, hipStream_t stream) {
  hipError_t e;
  switch (dpad) {
    case 32: e = launch_extend_rows<BF16, 32>(p, (int)l.items, stream); break;
    case 64: e = launch_extend_rows<BF16, 64>(p, (int)l.items, stream); break;
    case 128: e = launch_extend_rows<BF16, 128>(p, (int)l.items, stream); break;
    default: e = launch_extend_rows<BF16, 256>(p, (int)l.items, stream); break;
  }
  if (e != hipSuccess) return fail(FGW_MHA_EHIP, "fgw_kv_extend: %s", hipGetErrorString(e));
  if (l.target > 0) {
    const int64_t rows = std::min<int64_t>(kRowsTile, (int64_t)std::min(p.max_new, p.tokens) * p.group);
    extend_join_kernel<BF16, kRowsTile, kRowsBlock, true>
        <<<dim3((unsigned)(l.tiles * p.heads), (unsigned)rows), dim3(kMergeThreads), 0, stream>>>(
            p, p.lengths, p.cu);
    return launched("fgw_kv_extend");
  }
  return FGW_MHA_OK;
}

}  // namespace fgw_kv

using namespace fgw_kv;

extern "C" {

int fgw_kv_extend_workspace(const fgw_kv_extend_args* args, int64_t* floats) {
  if (int rc = check(args)) return rc;
  *floats = args->tokens == 0 ? 0 : plan_rows(*args).floats;
  return FGW_MHA_OK;
}

int fgw_kv_extend(const fgw_kv_extend_args* args, hipStream_t stream) {
  if (int rc = check(args)) return rc;
  const fgw_kv_extend_args& a = *args;
  if (a.tokens == 0) return FGW_MHA_OK;
  if (!a.q.data || !a.out || !a.k_cache || !a.v_cache || !a.block_table || !a.cache_seqlens || !a.cu_seqlens)
    return fail(FGW_MHA_EINVAL, "tensors are missing");
  if (!aligned16(a.q.data) || !aligned16(a.out) || !aligned16(a.k_cache) || !aligned16(a.v_cache) ||
      a.q.token_stride % 8 || a.q.head_stride % 8)
    return fail(FGW_MHA_EINVAL, "rows must be 16-byte aligned, their strides multiples of 16 bytes");
  const Launch l = plan_rows(a);
  if (l.items > 0x7fffffff) return fail(FGW_MHA_EUNSUPPORTED, "too many rows for one call");
  if (l.floats > 0 && (!a.workspace || !aligned16(a.workspace)))
    return fail(FGW_MHA_EINVAL, "the workspace is missing");
  ExtendParams p = {};
  p.q = a.q.data;
  p.q_token = a.q.token_stride * 2;
  p.q_head = a.q.head_stride * 2;
  p.k = a.k_cache;
  p.v = a.v_cache;
  p.table = a.block_table;
  p.lengths = a.cache_seqlens;
  p.cu = a.cu_seqlens;
  p.out = a.out;
  p.parts = a.workspace;
  p.lse = a.workspace ? a.workspace + l.items * l.rows_tile * a.dim : nullptr;
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
  p.window = a.window;
  p.rows_from = 0;
  p.rows_to = 0x7fffffff;
  p.work = (int)l.items;
  p.target = l.target;
  p.min_chunk = l.min_chunk;
  return a.dtype == FGW_KV_BFLOAT16 ? run_rows<true>(p, l, dim_tile(a.dim), stream)
                                    : run_rows<false>(p, l, dim_tile(a.dim), stream);
}

}  // extern "C"
