// Rotary positions, alone and on the way into the paged cache (fgw_rotary_apply, fgw_kv_append).
//
// Pair (a, b) of a row at position p: a' = s (a cos t - b sin t), b' = s (b cos t + a sin t) with
// t = p w. The frequency comes as a 64-bit fraction of a turn per position, so p w modulo a turn is
// one integer product that drops its high bits: exact at any position, where t in fp32 has lost
// its digits from some ten thousand positions on. The fraction is cut to an eighth of a turn
// either side of a quarter before it becomes fp32; on that range the Taylor series of sine (to
// x^9) and cosine (to x^10) are below fp32's rounding. Products and sums are fp32, rounded once.
//
// Both operators move their bytes once and are bound by that, or by latency for few tokens. A
// thread owns one unit of a token's heads, 16 bytes (both halves of the pairs in the half layout,
// so 32) at the same place of heads g, g + G, ...: it computes the unit's angles once and walks
// the heads. Neighbouring lanes own neighbouring units, then heads, so a wave reads whole rows.
// Heads per thread (per_thread): 1 while the threads do not fill the card, 2 beyond.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "fmha_kernel.h"
#include "kv_common.h"

namespace fgw_kv {

using fgw_mha::Elem;
using fgw_mha::u32;
using fgw_mha::u32x4;

constexpr int kThreads = 256;
constexpr int kLdsBatch = 1024;  // requests whose offsets a workgroup keeps in LDS

struct Rows {
  char* data;
  int64_t token, head;  // bytes
};

struct RotaryParams {
  Rows q, q_out, k, v;
  char* k_cache;
  char* v_cache;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* cu;
  const void* positions;
  const uint64_t* turns;
  int64_t pool_rows;
  int32_t positions64, tokens, batch, heads, kv_heads, width, page;
  u32 page_magic, page_shift;
  int32_t dim, rot, inverse;
  float scale;
  int32_t units;     // of a head
  int32_t rotating;  // units that hold pairs; the others copy 16 bytes
  int32_t groups;    // threads along the heads of a token
};

// 16 bytes of a row as fp32. KIND: fgw_kv_dtype.
template <int KIND>
constexpr int kPerChunk = KIND == FGW_KV_FLOAT32 ? 4 : 8;

template <int KIND>
__device__ __forceinline__ void unpack(u32x4 x, float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const u32 w = x[i];
    if constexpr (KIND == FGW_KV_FLOAT32) {
      f[i] = __uint_as_float(w);
    } else if constexpr (KIND == FGW_KV_BFLOAT16) {
      f[2 * i] = __uint_as_float(w << 16);
      f[2 * i + 1] = __uint_as_float(w & 0xffff0000u);
    } else {
      const fgw_mha::f16x2 h = __builtin_bit_cast(fgw_mha::f16x2, w);
      f[2 * i] = (float)h[0];
      f[2 * i + 1] = (float)h[1];
    }
  }
}

template <int KIND>
__device__ __forceinline__ u32x4 pack(const float* f) {
  u32x4 x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (KIND == FGW_KV_FLOAT32)
      x[i] = __float_as_uint(f[i]);
    else
      x[i] = Elem<KIND == FGW_KV_BFLOAT16>::pack2(f[2 * i], f[2 * i + 1]);
  }
  return x;
}

// 16 bytes of a row. Alone (ONCE) the rows pass the caches by: 268 MB in and out take 44 us, with ordinary
// loads 49, with non-temporal stores too 46; on the way into the pages 70 MB take 16 us with ordinary
// loads, 19 with these.
template <bool ONCE>
__device__ __forceinline__ u32x4 load_row(const char* at) {
  if constexpr (ONCE) return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(at));
  return fgw_mha::load16(at);
}

// scale cos and scale sin of turns * pos / 2^64 of a turn. The fraction is split into quarters
// rounded to nearest and a rest of at most an eighth (x = 2 pi rest, |x| <= pi / 4).
__device__ __forceinline__ void turn(uint64_t turns, uint64_t pos, float scale, float& c, float& s) {
  const uint64_t ph = turns * pos + (1ull << 61);
  const int quarter = (int)(ph >> 62);
  const int64_t rest = (int64_t)(ph & ((1ull << 62) - 1)) - (int64_t)(1ull << 61);
  const float x = (float)(int32_t)(rest >> 30) * 3.6572951981e-10f;  // 2 pi / 2^34
  const float z = x * x;
  float sn = __builtin_fmaf(z, 2.75573192e-6f, -1.98412698e-4f);
  sn = __builtin_fmaf(z, sn, 8.33333333e-3f);
  sn = __builtin_fmaf(z, sn, -1.66666667e-1f);
  sn = __builtin_fmaf(x * z, sn, x);
  float cs = __builtin_fmaf(z, -2.75573192e-7f, 2.48015873e-5f);
  cs = __builtin_fmaf(z, cs, -1.38888889e-3f);
  cs = __builtin_fmaf(z, cs, 4.16666667e-2f);
  cs = __builtin_fmaf(z, cs, -0.5f);
  cs = __builtin_fmaf(z, cs, 1.0f);
  const float a = quarter & 1 ? sn : cs, b = quarter & 1 ? cs : sn;
  c = scale * (quarter == 1 || quarter == 2 ? -a : a);
  s = scale * (quarter >= 2 ? -b : b);
}

// The request of a packed row: the last b with cu[b] <= t (cu[0] = 0, t < cu[batch]).
template <class P>
__device__ __forceinline__ int request_of(P cu, int batch, int t) {
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

template <int KIND, bool INTERLEAVED, bool APPEND>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryParams p) {
  constexpr int E = kPerChunk<KIND>;
  constexpr int NP = INTERLEAVED ? E / 2 : E;  // pairs of a unit
  __shared__ int32_t cu_lds[kLdsBatch + 1];
  if constexpr (APPEND) {
    if (p.batch <= kLdsBatch) {
      for (int i = threadIdx.x; i <= p.batch; i += kThreads) cu_lds[i] = p.cu[i];
      __syncthreads();
    }
  }
  const u32 id = blockIdx.x * kThreads + threadIdx.x;  // below 2^32 (layout)
  const u32 per_token = (u32)(p.units * p.groups);
  const u32 token = id / per_token;
  if (token >= (u32)p.tokens) return;
  const int t = (int)token, in_token = (int)(id - token * per_token);
  const int group = in_token / p.units, unit = in_token - group * p.units;
  const bool rotates = unit < p.rotating;

  int64_t pos = 0, row = -1;
  if constexpr (APPEND) {
    int b, first, next;
    if (p.batch <= kLdsBatch) {
      if (t >= cu_lds[p.batch]) return;
      b = request_of(cu_lds, p.batch, t);
      first = cu_lds[b];
      next = cu_lds[b + 1];
    } else {
      if (t >= p.cu[p.batch]) return;
      b = request_of(p.cu, p.batch, t);
      first = p.cu[b];
      next = p.cu[b + 1];
    }
    const int at = p.lens[b] - (next - first) + (t - first);
    pos = at;
    const u32 pg = fgw_mha::div_page((u32)at, p.page_magic, p.page_shift);
    if (at >= 0 && pg < (u32)p.width) {
      row = (int64_t)p.table[(int64_t)b * p.width + pg] * p.page + ((u32)at - pg * (u32)p.page);
      if (row >= p.pool_rows) row = -1;
    }
  }
  if (p.positions)
    pos = p.positions64 ? static_cast<const int64_t*>(p.positions)[t]
                        : (int64_t) static_cast<const int32_t*>(p.positions)[t];

  // The unit's chunks: bytes lo and hi of a head.
  const int lo = rotates ? unit * 16
                         : (p.rot + (unit - p.rotating) * E) * (16 / E);
  const int hi = lo + p.rot / 2 * (16 / E);
  float c[NP], s[NP];
  if (rotates) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      turn(p.turns[unit * NP + i], (uint64_t)pos, p.scale, c[i], s[i]);
      if (p.inverse) s[i] = -s[i];
    }
  }
  const int total = APPEND ? p.heads + 2 * p.kv_heads : p.heads;
  const int64_t pool_head = (int64_t)p.dim * (16 / E);
  auto step = [&](int head) {
    const char* src;
    char* dst;
    bool plain = !rotates;
    if (!APPEND || head < p.heads) {
      src = p.q.data + (int64_t)t * p.q.token + head * p.q.head;
      dst = p.q_out.data + (int64_t)t * p.q_out.token + head * p.q_out.head;
    } else {
      if (row < 0) return;
      const bool is_v = head >= p.heads + p.kv_heads;
      const int h = head - p.heads - (is_v ? p.kv_heads : 0);
      const Rows& x = is_v ? p.v : p.k;
      src = x.data + (int64_t)t * x.token + h * x.head;
      dst = (is_v ? p.v_cache : p.k_cache) + (row * p.kv_heads + h) * pool_head;
      plain |= is_v;
    }
    const u32x4 xa = load_row<!APPEND>(src + lo);
    if (!rotates) {
      *reinterpret_cast<u32x4*>(dst + lo) = xa;
      return;
    }
    if constexpr (INTERLEAVED) {
      float f[E], g[E];
      unpack<KIND>(xa, f);
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        g[2 * i] = f[2 * i] * c[i] - f[2 * i + 1] * s[i];
        g[2 * i + 1] = f[2 * i + 1] * c[i] + f[2 * i] * s[i];
      }
      *reinterpret_cast<u32x4*>(dst + lo) = plain ? xa : pack<KIND>(g);
    } else {
      const u32x4 xb = load_row<!APPEND>(src + hi);
      float f[E], g[E], u[E], w[E];
      unpack<KIND>(xa, f);
      unpack<KIND>(xb, g);
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        u[i] = f[i] * c[i] - g[i] * s[i];
        w[i] = g[i] * c[i] + f[i] * s[i];
      }
      *reinterpret_cast<u32x4*>(dst + lo) = plain ? xa : pack<KIND>(u);
      *reinterpret_cast<u32x4*>(dst + hi) = plain ? xb : pack<KIND>(w);
    }
  };
  for (int head = group; head < total; head += p.groups) step(head);
}

template <int KIND, bool APPEND>
void launch_rotary(const RotaryParams& p, bool interleaved, int64_t blocks, hipStream_t stream) {
  const dim3 grid((unsigned)blocks), threads(kThreads);
  if (interleaved)
    rotary_kernel<KIND, true, APPEND><<<grid, threads, 0, stream>>>(p);
  else
    rotary_kernel<KIND, false, APPEND><<<grid, threads, 0, stream>>>(p);
}

// Heads that one thread walks: enough threads for the card (256 CUs of 2048) come first. More than two
// leave fewer loads in flight than the memory takes (16384 tokens of 32 heads, D 128, us, at most 1 / 2 /
// 4 / 8 heads: 52 / 49 / 54 / 57, ordinary loads).
static int per_thread(int64_t units, int64_t tokens, int heads) {
  const int64_t n = units * tokens * heads / (256 * 2048);
  return n < 2 ? 1 : 2;
}

static int check_rotary(const fgw_kv_rotary& r, int dim) {
  if (r.dim <= 0 || r.dim % 16 || r.dim > dim)
    return fail(FGW_MHA_EINVAL, "rotated dims must be a positive multiple of 16, at most the head dim");
  if (!r.turns) return fail(FGW_MHA_EINVAL, "rotary frequencies are missing");
  return FGW_MHA_OK;
}

static bool rows_ok(const fgw_kv_rows& x, int elem, Rows& out) {
  if (!x.data || !aligned16(x.data) || (x.token_stride * elem) % 16 || (x.head_stride * elem) % 16)
    return false;
  out.data = static_cast<char*>(const_cast<void*>(x.data));
  out.token = x.token_stride * elem;
  out.head = x.head_stride * elem;
  return true;
}

// Units, groups and the grid of a launch; -1 when its threads would not count in 32 bits.
static int64_t layout(RotaryParams& p, bool interleaved, int elem, int heads) {
  const int per_chunk = 16 / elem;
  p.rotating = interleaved ? p.rot / per_chunk : p.rot / 2 / per_chunk;
  p.units = p.rotating + (p.dim - p.rot) / per_chunk;
  const int walk = per_thread(p.units, p.tokens, heads);
  p.groups = (heads + walk - 1) / walk;
  const int64_t blocks = ((int64_t)p.tokens * p.units * p.groups + kThreads - 1) / kThreads;
  return blocks < (1ll << 32) / kThreads ? blocks : -1;
}

}  // namespace fgw_kv

using namespace fgw_kv;

extern "C" {

int fgw_rotary_apply(const fgw_rotary_args* a, hipStream_t stream) {
  if (!a) return fail(FGW_MHA_EINVAL, "arguments are missing");
  if (a->dtype < FGW_KV_FLOAT16 || a->dtype > FGW_KV_FLOAT32)
    return fail(FGW_MHA_EUNSUPPORTED, "FP16, BF16 or FP32 rows required");
  if (a->dim <= 0 || a->dim % 16 || a->dim > 1024)
    return fail(FGW_MHA_EUNSUPPORTED, "the head dim must be in [16, 1024] and divisible by 16");
  if (a->tokens < 0 || a->heads <= 0) return fail(FGW_MHA_EINVAL, "positive extents required");
  if (int rc = check_rotary(a->rotary, a->dim)) return rc;
  if (a->tokens == 0) return FGW_MHA_OK;
  const int elem = a->dtype == FGW_KV_FLOAT32 ? 4 : 2;
  RotaryParams p = {};
  if (!rows_ok(a->x, elem, p.q) || !rows_ok(a->out, elem, p.q_out))
    return fail(FGW_MHA_EINVAL, "rows must be 16-byte aligned, their strides multiples of 16 bytes");
  if (!a->positions) return fail(FGW_MHA_EINVAL, "positions are missing");
  p.positions = a->positions;
  p.positions64 = a->positions64;
  p.turns = a->rotary.turns;
  p.tokens = a->tokens;
  p.heads = a->heads;
  p.dim = a->dim;
  p.rot = a->rotary.dim;
  p.inverse = a->rotary.inverse;
  p.scale = a->rotary.scale;
  const bool inter = a->rotary.interleaved != 0;
  const int64_t blocks = layout(p, inter, elem, p.heads);
  if (blocks < 0) return fail(FGW_MHA_EUNSUPPORTED, "too many rows for one call");
  if (a->dtype == FGW_KV_FLOAT32)
    launch_rotary<FGW_KV_FLOAT32, false>(p, inter, blocks, stream);
  else if (a->dtype == FGW_KV_BFLOAT16)
    launch_rotary<FGW_KV_BFLOAT16, false>(p, inter, blocks, stream);
  else
    launch_rotary<FGW_KV_FLOAT16, false>(p, inter, blocks, stream);
  return launched("fgw_rotary_apply");
}

int fgw_kv_append(const fgw_kv_append_args* a, hipStream_t stream) {
  if (!a) return fail(FGW_MHA_EINVAL, "arguments are missing");
  if (a->dtype != FGW_KV_FLOAT16 && a->dtype != FGW_KV_BFLOAT16)
    return fail(FGW_MHA_EUNSUPPORTED, "matching FP16/BF16 Q/K/V required");
  if (a->dim < 16 || a->dim > 256 || a->dim % 16)
    return fail(FGW_MHA_EUNSUPPORTED, "D must be in [16, 256] and divisible by 16");
  if (a->page_size <= 0 || a->pool_rows <= 0 || a->pool_rows % a->page_size || a->width <= 0)
    return fail(FGW_MHA_EINVAL,
                "positive page size, whole pool pages and positive table width required");
  if ((int64_t)a->width * a->page_size > 0x7fffffff)
    return fail(FGW_MHA_EUNSUPPORTED, "table capacity must fit in 31 bits");
  if (a->tokens < 0 || a->batch <= 0 || a->heads <= 0 || a->kv_heads <= 0)
    return fail(FGW_MHA_EINVAL, "positive extents required");
  const bool rotate = a->rotary.turns != nullptr;
  if (rotate) {
    if (int rc = check_rotary(a->rotary, a->dim)) return rc;
  }
  if (a->tokens == 0) return FGW_MHA_OK;
  RotaryParams p = {};
  if (!rows_ok(a->q, 2, p.q) || !rows_ok(a->q_out, 2, p.q_out) || !rows_ok(a->k, 2, p.k) ||
      !rows_ok(a->v, 2, p.v) || !aligned16(a->k_cache) || !aligned16(a->v_cache))
    return fail(FGW_MHA_EINVAL, "rows must be 16-byte aligned, their strides multiples of 16 bytes");
  if (!a->k_cache || !a->v_cache || !a->block_table || !a->cache_seqlens || !a->cu_seqlens)
    return fail(FGW_MHA_EINVAL, "tensors are missing");
  p.k_cache = static_cast<char*>(a->k_cache);
  p.v_cache = static_cast<char*>(a->v_cache);
  p.table = a->block_table;
  p.lens = a->cache_seqlens;
  p.cu = a->cu_seqlens;
  p.positions = a->positions;
  p.positions64 = a->positions64;
  p.turns = a->rotary.turns;
  p.pool_rows = a->pool_rows;
  p.tokens = a->tokens;
  p.batch = a->batch;
  p.heads = a->heads;
  p.kv_heads = a->kv_heads;
  p.width = a->width;
  p.page = a->page_size;
  page_division((uint32_t)a->page_size, p.page_magic, p.page_shift);
  p.dim = a->dim;
  p.rot = rotate ? a->rotary.dim : 0;
  p.inverse = a->rotary.inverse;
  p.scale = a->rotary.scale;
  const bool inter = rotate && a->rotary.interleaved != 0;
  const int64_t blocks = layout(p, inter, 2, p.heads + 2 * p.kv_heads);
  if (blocks < 0) return fail(FGW_MHA_EUNSUPPORTED, "too many rows for one call");
  if (a->dtype == FGW_KV_BFLOAT16)
    launch_rotary<FGW_KV_BFLOAT16, true>(p, inter, blocks, stream);
  else
    launch_rotary<FGW_KV_FLOAT16, true>(p, inter, blocks, stream);
  return launched("fgw_kv_append");
}

}  // extern "C"
