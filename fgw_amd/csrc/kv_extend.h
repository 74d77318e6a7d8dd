// Attention of packed new tokens over the paged cache, grouped K/V heads (fgw_kv_extend).
//
// Request b has n_b new tokens, the last of its len_b cached ones; query head h reads K/V head
// h / G, G = heads / kv_heads. The G query heads of a token that share a K/V head are rows of one
// tile: row R of (request, K/V head) is token R / G, head R % G of the group, so a tile of 32 rows
// reads each key once for all of them. Row R sees the keys [lo, hi) of its token:
//   hi = len - n + token + 1 (causal; else len),  lo = hi - window (no window: 0).
// Softmax and products are those of fmha_kernel.h (fp32 sums and statistics, P rounded to the
// input type for the PV product).
//
// Work. Lengths and counts are on the device, so the programs make the plan themselves (find_item):
// each reads the lengths of 64 requests at a time, one to a lane, and sums tiles and key blocks
// over the wave. W = kv_heads * sum(tiles * blocks) block visits; with `target` programs to fill
// the card a tile's keys are cut into ceil(blocks / chunk) splits, chunk = max(min_chunk, W /
// target): long requests into many, short ones not at all, and never more than target + tiles *
// kv_heads items in all, which bounds grid and workspace on the host without the lengths. The
// surplus programs end after the sums. Split tiles go through partials (O / l, LSE) and a join.
// Item w = ((request, tile, split), K/V head), the head fastest: workgroup w runs on XCD w % 8, so
// with 8 heads an XCD holds one of them, and every XCD has its share of every request.
#pragma once
#include "fmha_kernel.h"

namespace fgw_kv {

using namespace fgw_mha;

// heads: K/V heads; work: items of the launch at most; sq, q_tiles, mode, splits: unused.
struct ExtendParams : FwdParams {
  const int32_t* cu;
  int64_t q_token, q_head;  // bytes
  int32_t tokens, q_heads, group, max_new, window;
  int32_t rows_from, rows_to;  // requests with n * group in (rows_from, rows_to] are this launch's
  int32_t target, min_chunk;   // target 0: nothing is split
};

struct Request {
  int first, n, len, tiles, blocks;
};

template <int ROWS, int BN>
__device__ __forceinline__ Request load_request(const ExtendParams& p, const int32_t* lengths,
                                                const int32_t* cu, int b) {
  Request r{0, 0, 0, 0, 0};
  if (b >= p.batch) return r;
  const int first = cu[b], next = cu[b + 1];
  int len = lengths[b];
  const int capacity = p.width * p.page_size;
  r.len = len < 0 ? 0 : (len > capacity ? capacity : len);
  r.first = first;
  if (first < 0 || next > p.tokens || next <= first) return r;
  r.n = next - first < p.max_new ? next - first : p.max_new;
  const int64_t rows = (int64_t)r.n * p.group;
  if (rows <= p.rows_from || rows > p.rows_to) return r;
  r.tiles = (int)((rows + ROWS - 1) / ROWS);
  int lo = p.window > 0 ? r.len - r.n - p.window + 1 : 0;
  lo = lo < 0 ? 0 : lo;
  r.blocks = (r.len + BN - 1) / BN - lo / BN;
  return r;
}

// One item: tile `tile` of request `b`, split `split` of `splits`; its keys are the blocks
// [blk_begin, blk_end) and of those the keys [lo, hi) that some row of the tile sees.
struct Item {
  int b, first, n, len, tile, head, split, splits;
  int rows;                  // of the tile
  int lo, hi;
  int blk_begin, blk_end;
  int slot, slot_step;       // partials of split s: slot0 + s * slot_step; slot is this split's
};

__device__ __forceinline__ int wave_incl_sum(int x, int lane) {
  for (int off = 1; off < 64; off <<= 1) {
    const int up = __shfl_up(x, off, 64);
    x += lane >= off ? up : 0;
  }
  return x;
}

// Item w (BY_TILE: the first split of tile w / kv_heads, head w % kv_heads) of the launch; false
// past the last one. Uniform over the wave; every wave of a workgroup computes the same.
template <int ROWS, int BN, bool BY_TILE>
__device__ __forceinline__ bool find_item(const ExtendParams& p, const int32_t* lengths,
                                          const int32_t* cu, int w, int lane, Item& it) {
  const Request r0 = load_request<ROWS, BN>(p, lengths, cu, lane);
  int chunk = 0x40000000;
  if (p.target > 0) {
    float visits = 0.0f;  // (the same order in every program: the same sum)
    for (int b0 = 0; b0 < p.batch; b0 += 64) {
      const Request r = b0 == 0 ? r0 : load_request<ROWS, BN>(p, lengths, cu, b0 + lane);
      visits += (float)r.tiles * (float)r.blocks;
    }
#pragma unroll
    for (int x = 1; x < 64; x *= 2) visits += __shfl_xor(visits, x, 64);
    // (The bound on the items allows for the rounding of this sum: items_bound.)
    const float per = ceilf(visits * (float)p.heads / (float)p.target);
    chunk = per < 1.0e9f ? (int)per : 1000000000;
    chunk = __builtin_amdgcn_readfirstlane(chunk < p.min_chunk ? p.min_chunk : chunk);
  }
  const int g = w / p.heads;
  it.head = w - g * p.heads;
  int tiles_before = 0, items_before = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 64) {
    const Request r = b0 == 0 ? r0 : load_request<ROWS, BN>(p, lengths, cu, b0 + lane);
    const int splits = r.blocks > chunk ? (r.blocks + chunk - 1) / chunk : 1;
    const int items = r.tiles * splits;
    const int items_to = wave_incl_sum(items, lane);
    const int tiles_to = BY_TILE ? wave_incl_sum(r.tiles, lane) : 0;
    const int own = BY_TILE ? r.tiles : items;
    const int at = BY_TILE ? g - tiles_before - (tiles_to - own) : g - items_before - (items_to - own);
    const uint64_t hit = __ballot(at >= 0 && at < own);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      auto pick = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
      const int s = pick(splits), place = pick(at), tiles = pick(r.tiles);
      it.b = b0 + l;
      it.first = pick(r.first);
      it.n = pick(r.n);
      it.len = pick(r.len);
      // The last tiles first: causal, they are the longest.
      const int place_tile = BY_TILE ? place : place / s;
      it.tile = tiles - 1 - place_tile;
      it.split = BY_TILE ? 0 : place - place_tile * s;
      it.slot_step = p.heads;
      it.slot = (items_before + pick(items_to) - pick(items) + place_tile * s + it.split) * p.heads + it.head;

      const int row0 = it.tile * ROWS, all = it.n * p.group;
      it.rows = all - row0 < ROWS ? all - row0 : ROWS;
      const int t0 = row0 / p.group, t1 = (row0 + it.rows - 1) / p.group;
      int hi = p.causal ? it.len - it.n + t1 + 1 : it.len;
      hi = hi < 0 ? 0 : hi;
      int lo = p.window > 0 ? it.len - it.n + t0 - p.window + 1 : 0;
      lo = lo < 0 ? 0 : (lo > hi ? hi : lo);
      it.lo = lo;
      it.hi = hi;
      const int from = lo / BN, blocks = (hi + BN - 1) / BN - from;
      const int most = blocks > chunk ? (blocks + chunk - 1) / chunk : 1;
      it.splits = most < s ? most : s;
      it.blk_begin = from + split_bound(blocks, it.split, it.splits);
      it.blk_end = from + split_bound(blocks, it.split + 1, it.splits);
      return it.split < it.splits;
    }
    items_before += __shfl(items_to, 63, 64);
    if (BY_TILE) tiles_before += __shfl(tiles_to, 63, 64);
  }
  return false;
}

// The keys that row R of an item's tile sees.
struct Seen {
  int lo, hi;
};
__device__ __forceinline__ Seen row_seen(const ExtendParams& p, const Item& it, int token) {
  int hi = p.causal ? it.len - it.n + token + 1 : it.len;
  hi = hi < 0 ? 0 : hi;
  int lo = p.window > 0 ? it.len - it.n + token - p.window + 1 : 0;
  lo = lo < 0 ? 0 : lo;
  return Seen{lo, hi};
}

template <class C>
__device__ __forceinline__ void mask_seen(f32x16 (&s)[C::ST], int pos0, const Seen& seen, int hh) {
#pragma unroll
  for (int t = 0; t < C::ST; ++t)
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      const int key = pos0 + 32 * t + 8 * (v >> 2) + 4 * hh + (v & 3);
      s[t][v] = key >= seen.hi || key < seen.lo ? -INFINITY : s[t][v];
      __builtin_amdgcn_sched_barrier(0);
    }
}

// Rows that few requests' tokens fill: 32 rows to a tile, four waves that each stream their own
// 32-key blocks of the item through LDS and meet at its end (the key layout of fwd_kernel, whose
// operand layouts and softmax these are).
//
// DMA: lane l (mod 32) resolves key l of the block through the table, one block ahead of its use,
// and the load instructions fetch their rows' offsets from those lanes, so any page size takes the
// same path. Keys outside [lo, hi), page ids outside the pool and dims past D read zeros.
template <class C>
__device__ __forceinline__ int32_t key_page(const ExtendParams& p, const int32_t* table_b, int pos) {
  const u32 pg = div_page((u32)pos, p.page_magic, p.page_shift), last = (u32)p.width - 1u;
  return table_b[pg < last ? pg : last];
}

template <class C>
__device__ __forceinline__ void issue_rows(const ExtendParams& p, const char* kb, const char* vb,
                                           int64_t row_bytes, int pos, int32_t page_id, int lo, int hi,
                                           unsigned char* stage, int lane) {
  const u32 dst = (u32)opaque_uniform((int)lds_address(stage));
  const u32 pg = div_page((u32)pos, p.page_magic, p.page_shift);
  const int64_t row = (int64_t)page_id * p.page_size + ((u32)pos - pg * (u32)p.page_size);
  const bool live = pos >= lo && pos < hi && row >= 0 && row < p.pool_rows;
  const int64_t off = live ? row * row_bytes : -1;
  const u32 off_lo = (u32)off, off_hi = (u32)((uint64_t)off >> 32);
  const char* zero = reinterpret_cast<const char*>(kZeroChunk);
#pragma unroll
  for (int i = 0; i < C::INSTR; ++i) {
    const int r = C::RPI * i + lane / C::CPR, at = lane % C::CPR;
    const u32 rl = (u32)__builtin_amdgcn_ds_bpermute(4 * r, (int)off_lo);
    const u32 rh = (u32)__builtin_amdgcn_ds_bpermute(4 * r, (int)off_hi);
    const int64_t ro = (int64_t)(((uint64_t)rh << 32) | rl);
    const int kc = at ^ (r % C::KSW), vc = at ^ (4 * (r % C::VSW));
    const char* ks = ro >= 0 && kc * 8 < p.dim ? kb + ro + kc * 16 : zero;
    const char* vs = ro >= 0 && vc * 8 < p.dim ? vb + ro + vc * 16 : zero;
    __builtin_amdgcn_global_load_lds(ks, FGW_LDS(void, (uintptr_t)(dst + 1024u * i)), 16, 0, 0);
    __builtin_amdgcn_global_load_lds(vs, FGW_LDS(void, (uintptr_t)(dst + C::TILE_BYTES + 1024u * i)), 16,
                                     0, 0);
  }
}

template <class C>
__global__ __launch_bounds__(C::THREADS) void extend_rows_kernel(ExtendParams p,
                                                                 const int32_t* __restrict__ table,
                                                                 const int32_t* __restrict__ lengths,
                                                                 const int32_t* __restrict__ cu) {
  constexpr int kBytes = CMax<C::TILES_BYTES, C::COMB_BYTES>::value;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[kBytes];
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int il = lane & 31, hh = lane >> 5;
  Item it;
  if (!find_item<C::ROWS_TILE, C::BN, false>(p, lengths, cu, (int)blockIdx.x, lane, it)) return;

  const Lanes<C> ln(lane);
  const int64_t row_bytes = (int64_t)p.heads * p.dim * 2;
  const int32_t* table_b = table + (int64_t)it.b * p.width;
  const char* kb = static_cast<const char*>(p.k) + (int64_t)it.head * p.dim * 2;
  const char* vb = static_cast<const char*>(p.v) + (int64_t)it.head * p.dim * 2;
  unsigned char* const stages = smem + wave * C::GROUP_BYTES;

  // This wave's blocks: blk_begin + wave, + 4, ...
  constexpr int kStep = C::NWK * C::BN;
  const int cnt = it.blk_end - it.blk_begin;
  const int my_n = cnt > wave ? (cnt - wave + C::NWK - 1) / C::NWK : 0;
  const int first_pos = (it.blk_begin + wave) * C::BN;
  int32_t id = my_n > 0 ? key_page<C>(p, table_b, first_pos + il) : 0;
  int32_t next_id = my_n > 1 ? key_page<C>(p, table_b, first_pos + kStep + il) : 0;
  if (my_n > 0)
    issue_rows<C>(p, kb, vb, row_bytes, first_pos + il, id, it.lo, it.hi, stages, lane);

  const int row = it.tile * C::ROWS_TILE + il;
  const int token = row / p.group, in_group = row - token * p.group;
  const bool mine = il < it.rows;
  u32x4 qf[C::KK];
  {
    const char* qp = static_cast<const char*>(p.q) + (int64_t)(it.first + token) * p.q_token +
                     (int64_t)(it.head * p.group + in_group) * p.q_head;
#pragma unroll
    for (int kk = 0; kk < C::KK; ++kk) {
      const int d = 16 * kk + 8 * hh;
      u32x4 val = {0u, 0u, 0u, 0u};
      if (mine && d < p.dim) val = load16(qp + 2 * d);
      qf[kk] = val;
    }
  }
  const Seen seen = row_seen(p, it, token);
  // Blocks with keys that some row of the tile does not see: past the first token's last key, or
  // below the last token's first.
  const int hi_min = row_seen(p, it, it.tile * C::ROWS_TILE / p.group).hi;
  const int lo_max = row_seen(p, it, (it.tile * C::ROWS_TILE + it.rows - 1) / p.group).lo;

  float m = kNegBig, l = 0.0f;
  f32x16 o[C::DT];
#pragma unroll
  for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[dt][v] = 0.0f;

  for (int n = 0; n < my_n; ++n) {
    const int pos0 = first_pos + kStep * n;
    unsigned char* stage = stages + (n % C::NBUF) * C::STAGE_BYTES;
    wait_dma();
    group_sync<C>();
    const int32_t id1 = next_id;
    if (n + 2 < my_n) next_id = key_page<C>(p, table_b, pos0 + 2 * kStep + il);
    if (n + 1 < my_n && C::NBUF == 2)
      issue_rows<C>(p, kb, vb, row_bytes, pos0 + kStep + il, id1, it.lo, it.hi,
                    stages + ((n + 1) % C::NBUF) * C::STAGE_BYTES, lane);
    f32x16 s[C::ST];
    u32x4 pf[C::KS];
    qk_block<C>(stage, ln, qf, s);
    if (pos0 + C::BN > hi_min || pos0 < lo_max) mask_seen<C>(s, pos0, seen, hh);
    online_softmax<C>(s, m, l, o, p.scale_log2, pf);
    pv_block<C>(stage + C::TILE_BYTES, ln, pf, o);
    if (n + 1 < my_n && C::NBUF == 1) {
      group_sync<C>();
      issue_rows<C>(p, kb, vb, row_bytes, pos0 + kStep + il, id1, it.lo, it.hi, stage, lane);
    }
  }
  wait_dma();

  // The waves' states of the same rows, through LDS.
  __syncthreads();
  float* cm = reinterpret_cast<float*>(smem);
  float* cl = cm + C::NWK * C::ROWS_WAVE;
  float* co = cl + C::NWK * C::ROWS_WAVE;
  const float tot = pair_sum(l);
  if (hh == 0) {
    cm[wave * C::ROWS_WAVE + il] = m;
    cl[wave * C::ROWS_WAVE + il] = tot;
  }
  if (mine) {
#pragma unroll
    for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
      for (int gq = 0; gq < 4; ++gq) {
        f32x4 val = {o[dt][4 * gq], o[dt][4 * gq + 1], o[dt][4 * gq + 2], o[dt][4 * gq + 3]};
        *reinterpret_cast<f32x4*>(co + (wave * C::ROWS_WAVE + il) * C::OSTRIDE + 32 * dt + 8 * gq +
                                  4 * hh) = val;
      }
  }
  __syncthreads();
  using E = Elem<C::BF16>;
  constexpr int D4 = C::DPAD / 4;
  for (int idx = tid; idx < it.rows * D4; idx += C::THREADS) {
    const int r = idx / D4, d0 = 4 * (idx % D4);
    if (d0 >= p.dim) continue;
    float mm = kNegBig;
#pragma unroll
    for (int k = 0; k < C::NWK; ++k) mm = fmaxf(mm, cm[k * C::ROWS_WAVE + r]);
    float t2 = 0.0f;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < C::NWK; ++k) {
      const float wt = __builtin_amdgcn_exp2f(cm[k * C::ROWS_WAVE + r] - mm);
      t2 += cl[k * C::ROWS_WAVE + r] * wt;
      acc += *reinterpret_cast<const f32x4*>(co + (k * C::ROWS_WAVE + r) * C::OSTRIDE + d0) * wt;
    }
    const float inv = 1.0f / fmaxf(t2, 1.0e-30f);
    if (it.splits == 1) {
      const int rr = it.tile * C::ROWS_TILE + r, tk = rr / p.group;
      u16* dst = static_cast<u16*>(p.out) +
                 ((int64_t)(it.first + tk) * p.q_heads + it.head * p.group + (rr - tk * p.group)) * p.dim + d0;
      u32x2 w;
      w.x = E::pack2(acc[0] * inv, acc[1] * inv);
      w.y = E::pack2(acc[2] * inv, acc[3] * inv);
      *reinterpret_cast<u32x2*>(dst) = w;
    } else {
      *reinterpret_cast<f32x4*>(p.parts + ((int64_t)it.slot * C::ROWS_TILE + r) * p.dim + d0) = acc * inv;
      if (d0 == 0) p.lse[(int64_t)it.slot * C::ROWS_TILE + r] = lse_of(mm, t2);
    }
  }
}

// The join of split tiles: workgroup (tile and head, part of its rows). D / 4 threads hold a row;
// the workgroup's kMergeThreads / (D / 4) such groups share a row's splits (WIDE: few rows, many
// splits) or take a row each. Weights exp(LSE - peak), empty splits (LSE -1e30) weigh nothing, an
// all-empty row is zero.
template <bool BF16, int ROWS, int BN, bool WIDE>
__global__ __launch_bounds__(kMergeThreads) void extend_join_kernel(ExtendParams p,
                                                                    const int32_t* __restrict__ lengths,
                                                                    const int32_t* __restrict__ cu) {
  using E = Elem<BF16>;
  __shared__ float speak[kMergeThreads], stot[kMergeThreads];
  __shared__ f32x4 sacc[kMergeThreads];
  const int t = threadIdx.x;
  Item it;
  if (!find_item<ROWS, BN, true>(p, lengths, cu, (int)blockIdx.x, t & 63, it)) return;
  // (Offsets that overlap make more items than the workspace has places for.)
  if (it.splits == 1 || (int64_t)it.slot + (int64_t)(it.splits - 1) * it.slot_step >= p.work) return;
  const int d4n = p.dim / 4, G = kMergeThreads / d4n;
  const int c = t % d4n, g = t / d4n;
  const int64_t ls = (int64_t)it.slot_step * ROWS;
  for (int r0 = blockIdx.y * (WIDE ? 1 : G); r0 < it.rows; r0 += gridDim.y * (WIDE ? 1 : G)) {
    const int r = WIDE ? r0 : r0 + g;
    const bool act = g < G && r < it.rows;
    const float* lse = p.lse + (int64_t)it.slot * ROWS + r;
    const float* parts = p.parts + ((int64_t)it.slot * ROWS + r) * p.dim + 4 * c;
    float peak = kNegBig, tot = 0.0f;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    if (act) wide_group<8>(lse, parts, ls, ls * p.dim, WIDE ? g : 0, WIDE ? G : 1, it.splits, peak, tot, acc);
    if constexpr (WIDE) {
      if (act && c == 0) speak[g] = peak;
      __syncthreads();
      float top = kNegBig;
      for (int k = 0; k < G; ++k) top = fmaxf(top, speak[k]);
      if (act) {
        const float scale = expf(peak - top);
        sacc[t] = acc * scale;
        if (c == 0) stot[g] = tot * scale;
      }
      __syncthreads();
      if (g == 0) {
        acc = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        tot = 0.0f;
        for (int k = 0; k < G; ++k) {
          acc += sacc[k * d4n + c];
          tot += stot[k];
        }
      }
    }
    if (act && (!WIDE || g == 0)) {
      const float inv = 1.0f / fmaxf(tot, 1.0e-30f);
      const int rr = it.tile * ROWS + r, tk = rr / p.group;
      u16* dst = static_cast<u16*>(p.out) +
                 ((int64_t)(it.first + tk) * p.q_heads + it.head * p.group + (rr - tk * p.group)) * p.dim + 4 * c;
      u32x2 w;
      w.x = E::pack2(acc[0] * inv, acc[1] * inv);
      w.y = E::pack2(acc[2] * inv, acc[3] * inv);
      *reinterpret_cast<u32x2*>(dst) = w;
    }
    if constexpr (WIDE) __syncthreads();  // the LDS entries are written again
  }
}

template <bool BF16, int DPAD>
hipError_t launch_extend_rows(const ExtendParams& p, int grid, hipStream_t stream) {
  using C = Cfg<BF16, DPAD, kLayoutKey, DPAD == 128 ? 1 : 0>;
  extend_rows_kernel<C><<<dim3(grid), dim3(C::THREADS), 0, stream>>>(p, p.table, p.lengths, p.cu);
  return hipGetLastError();
}

}  // namespace fgw_kv
