// C ABI of the attention over pages where groups of requests share a prefix (fgw_kv_shared).
//
// With the keys of a row cut in two, its prefix's and its own, and o, lse of each part alone,
//   w = exp(lse - max lse),  o = (w_prefix o_prefix + w_own o_own) / (w_prefix + w_own).
// Two passes of the kernels of fgw_kv_extend, each of which finds its requests on the device:
//   1. A group is one request: its rows are those of all its tokens (they lie side by side in q), its keys
//      the prefix, read through the first request's row of the table, with nothing to mask. Every item
//      leaves partials (O / l, LSE).
//   2. Each request over the keys behind its prefix; an unsplit tile takes the prefix's partials at its
//      end and writes the output, a split one's join takes them with its own.
// A request that does not reach past the prefix with all its new tokens, or is alone in its group, reads
// all its keys itself in the second pass.
//
// Where sharing pays. The passes cost a second launch, and partials of every row and split written and read; what
// they save is reading: requests of few rows read their keys once for every 32 of them. Requests of more
// than kShareRows rows are bound by products, of which there are as many either way. Shared / each on its own,
// us (requests x tokens, Hq 32, Hkv 8, D 128, reads saved): 8x1 prefix 3000 (98 MB) 23.4 / 19.7, 4096 (134 MB)
// 24.1 / 24.5, 16x1 2000 (131 MB) 24.7 / 24.6, 4096 (268 MB) 24.0 / 37.0, 32x1 8000 (1 GB) 35.1 / 106; 32x4 2000
// (262 MB) 37.2 / 35.2, 3000 (393 MB) 37.9 / 45.9; 32x8 3000 (393 MB) 49.6 / 46.8, 4096 (537 MB) 55.4 / 60.4; 64x8
// 4096 (1.1 GB) 79.5 / 77.4; 32x32 2000 (1 GB) 100.6 / 90.1, 3000 (1.6 GB) 119.1 / 120.1, 8192 (4.3 GB) 238 / 296;
// 8x64 16000 231 / 136, 8x512 4096 481 / 269. Hence 100 MB, and as much for the partials as 340 bytes for every dim
// of every row that shares. The device knows lengths and groups and decides; where the table's capacity rules it
// out, or tokens and requests do on average, the host leaves the first pass away (which costs 5 us where it is empty;
// how many of the call's rows share is not known there, and it counts 96 bytes for each).
#include <hip/hip_runtime.h>

#include "kv_extend_plan.h"

namespace fgw_kv {

#define FGW_KV_EXTERN(BF, P)                                                             \
  extern template hipError_t launch_extend_rows<BF, 32, P>(const P&, int, hipStream_t);  \
  extern template hipError_t launch_extend_rows<BF, 64, P>(const P&, int, hipStream_t);  \
  extern template hipError_t launch_extend_rows<BF, 128, P>(const P&, int, hipStream_t); \
  extern template hipError_t launch_extend_rows<BF, 256, P>(const P&, int, hipStream_t); \
  extern template hipError_t launch_extend_wide<BF, 256, P>(const P&, int, hipStream_t);
FGW_KV_EXTERN(true, PrefixParams) FGW_KV_EXTERN(true, SuffixParams)
FGW_KV_EXTERN(false, PrefixParams) FGW_KV_EXTERN(false, SuffixParams)
#define FGW_KV_EXTERN_WIDE(BF, DP) \
  extern template hipError_t launch_extend_wide<BF, DP, PrefixParams>(const PrefixParams&, int, hipStream_t);
FGW_KV_EXTERN_WIDE(true, 64) FGW_KV_EXTERN_WIDE(true, 128) FGW_KV_EXTERN_WIDE(false, 64) FGW_KV_EXTERN_WIDE(false, 128)
#define FGW_KV_EXTERN_LONG(BF, DP, R) \
  extern template hipError_t launch_extend_long<BF, DP, R, SuffixParams>(const SuffixParams&, int, hipStream_t);
#define FGW_KV_EXTERN_LONGS(BF)                                                                               \
  FGW_KV_EXTERN_LONG(BF, 64, kRowsBlock) FGW_KV_EXTERN_LONG(BF, 64, kRowsGroup) FGW_KV_EXTERN_LONG(BF, 64, kRowsPadded) \
  FGW_KV_EXTERN_LONG(BF, 128, kRowsBlock) FGW_KV_EXTERN_LONG(BF, 128, kRowsGroup) FGW_KV_EXTERN_LONG(BF, 128, kRowsPadded)
FGW_KV_EXTERN_LONGS(true) FGW_KV_EXTERN_LONGS(false)

namespace {

// The kernel of the first pass by the rows of a group: a short tile reads the keys for 32 of them, a wide one
// for 128. Both hold the weights of the PV product in two numbers of the input type, as few rows have them
// alone, so that what a token gets does not hang on who shares its prefix. Short / wide, us (Hq 32, Hkv 8, D
// 128): 48 rows, four prefixes of 4096 keys 36.0 / 36.6, one of 8192 64 rows 27.4 / 30.0; 80 rows, four of 4096
// 56.2 / 47.6, 128 rows 59.8 / 51.0. Wide with one number, two: 256 rows, one of 8192 36.0 / 38.6, 2048 of 4096
// 77 / 89, 4096 111 / 143. (Tiles of 256 rows with one number took 109.5 for the last.)
constexpr int kWideFrom = 64;
constexpr int kPrefixMinChunk = 2;  // blocks of 64 keys; 1 / 2 / 4, us: four prefixes of 1000 keys, 128 rows each 46.1 / 46.1 / 48.1
constexpr int64_t kShareBytes = 100 << 20, kHostDimBytes = 96;

struct SharedPlan {
  Launch prefix;
  int prefix_rows;  // of a place
  bool wide;        // the first pass's kernel
  int64_t notes;    // floats of the groups' notes
  Plan suffix;
  int share_from;   // SharedParams
};

template <class T>
void plan_prefix(SharedPlan& s, const fgw_kv_extend_args& a, int64_t groups) {
  Launch& l = s.prefix;
  const int64_t total = (int64_t)a.tokens * (a.heads / a.kv_heads);
  s.prefix_rows = T::ROWS;
  l.many = 1 << 20;
  l.tiles = total / T::ROWS + std::min<int64_t>(groups, a.tokens);
  plan_items<T>(l, a, true);
  l.slots = l.items;  // every item leaves partials
  l.floats = l.slots * T::ROWS * (a.dim + 1);
}

SharedPlan plan_shared(const fgw_kv_shared_args& args) {
  fgw_kv_extend_args a = args.attend;
  SharedPlan s = {};
  s.suffix = plan(a);
  if (args.groups == 0) return s;
  a.num_cus = std::min(a.num_cus, kMostCus);
  const int64_t total = (int64_t)a.tokens * (a.heads / a.kv_heads);
  if (!args.always) {
    const int64_t from = kShareBytes + kHostDimBytes * a.dim * a.heads * a.tokens;
    const int64_t requests = std::min(a.batch, a.tokens), key_bytes = 4 * (int64_t)a.kv_heads * shared_dims(a.dim);
    const double most = (double)(total / 32 + requests) * ((double)a.width * a.page_size) * (double)key_bytes;
    if (most < (double)from || total > (int64_t)kShareRows * requests) return s;
    s.share_from = (int)(kShareBytes >> 16);
  }
  const int64_t rows = total / args.groups;  // of a group, on average
  s.wide = rows > kWideFrom;
  s.prefix.min_chunk = s.wide ? kPrefixMinChunk : kRowsMinChunk;
  if (s.wide)
    plan_prefix<WideTiling>(s, a, args.groups);
  else
    plan_prefix<ShortTiling>(s, a, args.groups);
  s.notes = (int64_t)args.groups * (int64_t)sizeof(GroupNote) / 4;
  return s;
}

int check_shared(const fgw_kv_shared_args* args) {
  if (!args) return fail(FGW_MHA_EINVAL, "arguments are missing");
  if (int rc = check(&args->attend)) return rc;
  if (!args->attend.causal || args->attend.window != 0)
    return fail(FGW_MHA_EUNSUPPORTED, "attention with shared prefixes is causal and has no window");
  if (args->groups < 0) return fail(FGW_MHA_EINVAL, "the number of groups must not be negative");
  return FGW_MHA_OK;
}

template <bool BF16>
int run_shared(const fgw_kv_shared_args& args, const SharedPlan& s, hipStream_t stream) {
  const fgw_kv_extend_args& a = args.attend;
  SuffixParams own = params_of<SuffixParams>(a);
  float* work = a.workspace;
  own.groups = args.cu_groups;
  own.prefixes = args.prefix_lens;
  own.n_groups = s.prefix.items > 0 ? args.groups : 0;
  own.share_from = s.share_from;
  if (s.prefix.items > 0) {
    PrefixParams p = params_of<PrefixParams>(a);
    static_cast<SharedParams&>(p) = own;
    p.causal = 0;
    p.max_new = p.tokens;
    p.target = s.prefix.target;
    p.min_chunk = s.prefix.min_chunk;
    p.whole = s.prefix.whole;
    p.many = s.prefix.many;
    p.work = (int)s.prefix.slots;
    p.group_notes = reinterpret_cast<int32_t*>(work);
    p.parts = work + s.notes;
    p.lse = p.parts + s.prefix.slots * s.prefix_rows * a.dim;
    own.group_notes = p.group_notes;
    own.prefix_parts = p.parts;
    own.prefix_lse = p.lse;
    own.prefix_slots = p.work;
    own.prefix_rows = s.prefix_rows;
    work = p.parts + s.prefix.floats;
    const auto entry = !s.wide        ? rows_entry<BF16, PrefixParams>(a.dim)
                       : a.dim <= 64  ? &launch_extend_wide<BF16, 64, PrefixParams>
                       : a.dim <= 128 ? &launch_extend_wide<BF16, 128, PrefixParams>
                                      : &launch_extend_wide<BF16, 256, PrefixParams>;
    const hipError_t e = entry(p, (int)s.prefix.items, stream);
    if (e != hipSuccess) return fail(FGW_MHA_EHIP, "fgw_kv_shared: %s", hipGetErrorString(e));
  }
  own.parts = work;
  own.counters = s.suffix.rows.counters > 0 ? a.counters : nullptr;
  return run<BF16>(own, s.suffix, "fgw_kv_shared", stream);
}

}  // namespace

}  // namespace fgw_kv

using namespace fgw_kv;

extern "C" {

int fgw_kv_shared_workspace(const fgw_kv_shared_args* args, int64_t* floats, int64_t* counters) {
  if (int rc = check_shared(args)) return rc;
  *floats = *counters = 0;
  if (args->attend.tokens == 0) return FGW_MHA_OK;
  const SharedPlan s = plan_shared(*args);
  *floats = s.notes + s.prefix.floats + s.suffix.rows.floats + s.suffix.longs.floats;
  *counters = s.suffix.rows.counters;
  return FGW_MHA_OK;
}

int fgw_kv_shared(const fgw_kv_shared_args* args, hipStream_t stream) {
  if (int rc = check_shared(args)) return rc;
  const fgw_kv_extend_args& a = args->attend;
  if (a.tokens == 0) return FGW_MHA_OK;
  if (int rc = check_tensors(a)) return rc;
  if (args->groups > 0 && (!args->cu_groups || !args->prefix_lens)) return fail(FGW_MHA_EINVAL, "tensors are missing");
  const SharedPlan s = plan_shared(*args);
  if (std::max(s.prefix.items, std::max(s.suffix.rows.items, s.suffix.longs.items)) > 0x3fffffff)
    return fail(FGW_MHA_EUNSUPPORTED, "too many rows for one call");
  if (s.notes + s.prefix.floats + s.suffix.rows.floats + s.suffix.longs.floats > 0 && (!a.workspace || !aligned16(a.workspace)))
    return fail(FGW_MHA_EINVAL, "the workspace is missing");
  return a.dtype == FGW_KV_BFLOAT16 ? run_shared<true>(*args, s, stream) : run_shared<false>(*args, s, stream);
}

}  // extern "C"
