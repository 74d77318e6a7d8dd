// Long tiles of the attention over pages (fgw_kv_extend): 256 rows of (token, head of the group),
// eight waves that share every 64-key block of the item.
//
// The main loop is the one of prefill_kernel (fmha_prefill.h): two groups of four waves, one phase
// apart, so that on every SIMD one wave issues MFMAs while the other runs its softmax; K and V
// blocks come by DMA into rings of four slots, two blocks ahead. What differs: a program runs one
// item, found from the lengths on the device (find_item); a lane's row is a (token, head) pair, so
// its keys end at its own token and, with a window, begin at it; output rows are written by token.
// P is rounded once to the input type for the PV product (kv_extend.h gives the error and the cost of
// more). An item reads its keys once for the G heads of a group: at G 4 and 64 tokens a tile, a block of
// 32 KB feeds 4.3 MFLOP.
//
// ROWS as in fmha_prefill.h: blocks in one page (page_size a multiple of 64), row groups (a page
// table lookup per DMA instruction) and padded head dims. A block with keys outside the item's
// [lo, hi), or with a page outside the pool, is fetched key by key; those keys read zeros.
#pragma once
#include "fmha_prefill.h"
#include "kv_extend.h"

namespace fgw_kv {

// Pool byte offset of the first key of DMA unit u of the item (a block, or with row groups one
// instruction of this wave in a block), or -1 where it needs the lookup per key.
template <class C>
__device__ __forceinline__ int64_t unit_offset(const ExtendParams& p, const int32_t* table_b,
                                               int64_t row_bytes, int key0, int N, int lo, int hi, int j,
                                               int q, int wave) {
  constexpr bool kBlock = C::ROWS == kRowsBlock;
  constexpr int kKeys = kBlock ? C::BN : C::RPI;
  const int64_t at = (int64_t)key0 + (int64_t)j * C::BN + (kBlock ? 0 : C::RPI * (q * C::NWQ + wave));
  if (j >= N) return -1;
  const u32 pos0 = (u32)at;
  const u32 pg = div_page(pos0, p.page_magic, p.page_shift), last = (u32)p.width - 1u;
  const u32 in_page = pos0 - pg * (u32)p.page_size;
  const int32_t id = table_b[pg < last ? pg : last];
  const int64_t row0 = (int64_t)id * p.page_size + in_page;
  const bool fast = at >= lo && at + kKeys <= hi && in_page + kKeys <= (u32)p.page_size && row0 >= 0 &&
                    row0 + kKeys <= p.pool_rows && (C::ROWS != kRowsBlock || p.dim == C::DPAD);
  return fast ? row0 * row_bytes : -1;
}

template <class C>
__device__ __forceinline__ int64_t unit_window(const ExtendParams& p, const int32_t* table_b,
                                               int64_t row_bytes, int key0, int N, int lo, int hi, int w,
                                               int wave, int lane) {
  if constexpr (C::ROWS == kRowsBlock)
    return unit_offset<C>(p, table_b, row_bytes, key0, N, lo, hi, C::WINDOW * w + lane, 0, wave);
  else
    return unit_offset<C>(p, table_b, row_bytes, key0, N, lo, hi, C::WINDOW * w + lane / C::INSTR_PER_WAVE,
                          lane % C::INSTR_PER_WAVE, wave);
}

// DMA instruction q of this wave in the K (IS_V false) or V tile of the keys [pos0, pos0 + BN), each
// key through the table.
template <class C, bool IS_V>
__device__ __forceinline__ void issue_keys(const ExtendParams& p, const int32_t* table_b, const char* base,
                                           int64_t row_bytes, int pos0, int lo, int hi, u32 dst, int wave,
                                           int lane, int q) {
  const int dim = opaque_uniform(p.dim);
  lane = opaque_lane(lane);
  const char* zero = reinterpret_cast<const char*>(kZeroChunk);
  const int i = q * C::NWQ + wave;
  const int r = C::RPI * i + lane / C::CPR, at = lane % C::CPR;
  const int pos = pos0 + r;
  const bool in = pos >= lo && pos < hi;
  const u32 pg = in ? div_page((u32)pos, p.page_magic, p.page_shift) : 0u;
  const int64_t row = (int64_t)table_b[pg] * p.page_size + ((u32)pos - pg * (u32)p.page_size);
  const bool live = in && row >= 0 && row < p.pool_rows;
  const int c = IS_V ? at ^ (4 * (r % C::VSW)) : at ^ (r % C::KSW);
  dma_flat(live && c * 8 < dim ? base + row * row_bytes + c * 16 : zero, dst + 1024u * i);
}

// The 32 rows from `first_row` of an item's tile that one wave holds in o, m, l: to the output, or to
// the partials of a split tile, whole rows through the wave's LDS at `st` (32 kStagedRowBytes<C>).
template <class C>
__device__ __forceinline__ void store_wave_rows(const ExtendParams& p, const Item& it, int first_row,
                                                unsigned char* st, int lane, const f32x16 (&o)[C::DT], float m,
                                                float l) {
  const float tot = pair_sum(l), inv = 1.0f / fmaxf(tot, 1.0e-30f);
  const bool split = it.splits > 1;
  const int rows = it.rows - first_row;  // of this wave, where fewer than 32
  const int ln = opaque_lane(lane), lr = ln & 31, lh = ln >> 5;
  auto row_at = [&](int r) {
    return static_cast<u16*>(p.out) + out_row(p, it, it.tile * C::ROWS_TILE + first_row + r);
  };
  float* const parts = p.parts + ((int64_t)it.slot * C::ROWS_TILE + first_row) * p.dim;
  if (p.dim == C::DPAD) {
    if (split) {
      store_rows_staged<C>(st, lane, o, inv, true, parts, nullptr, 0, rows);
    } else {
      constexpr int NCH = C::DPAD * 2 / 16, RPS = 64 / NCH;
      write_staged_bf16<C>(st, lr, lh, o, inv);
#pragma unroll
      for (int k = 0; k < kStagedChunks<C>; ++k) {
        const int r = RPS * k + ln / NCH;
        const u32x4 v = read_staged_bf16<C>(st, ln, k);
        if (r < rows) __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(row_at(r) + 8 * (ln % NCH)));
      }
    }
  } else if (lr < rows) {
    using E = Elem<C::BF16>;
    u16* const dst = row_at(lr);
#pragma unroll
    for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
      for (int gq = 0; gq < 4; ++gq) {
        const int d0 = 32 * dt + 8 * gq + 4 * lh;
        if (d0 >= p.dim) continue;
        const f32x4 val = f32x4{o[dt][4 * gq], o[dt][4 * gq + 1], o[dt][4 * gq + 2], o[dt][4 * gq + 3]} * inv;
        if (split) {
          *reinterpret_cast<f32x4*>(parts + lr * p.dim + d0) = val;
        } else {
          *reinterpret_cast<u32x2*>(dst + d0) = u32x2{E::pack2(val[0], val[1]), E::pack2(val[2], val[3])};
        }
      }
  }
  if (split && lh == 0 && lr < rows) p.lse[(int64_t)it.slot * C::ROWS_TILE + first_row + lr] = part_lse(m, tot);
}

template <class C>
__global__ __attribute__((aligned(4096))) __launch_bounds__(C::THREADS) void extend_long_kernel(
    ExtendParams p, const int32_t* __restrict__ table, const int32_t* __restrict__ lengths,
    const int32_t* __restrict__ cu) {
  __shared__ __attribute__((aligned(1024))) unsigned char smem[C::RING_BYTES];
  const u32 kring_lds = lds_address(smem);
  const u32 vring_lds = kring_lds + (u32)(C::NKSLOT * C::TILE_BYTES);
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int il = lane & 31, hh = lane >> 5;
  Item it;
  const bool found = find_item<LongTiling>(p, lengths, cu, (int)blockIdx.x, lane, it);
  write_note(p, it, found);
  if (!found) return;

  const int64_t row_bytes = (int64_t)p.heads * p.dim * 2;
  const int32_t* table_b = table + (int64_t)it.b * p.width;
  const char* kb = static_cast<const char*>(p.k) + (int64_t)it.head * p.dim * 2;
  const char* vb = static_cast<const char*>(p.v) + (int64_t)it.head * p.dim * 2;
  const int key0 = it.blk_begin * C::BN, N = it.blk_end - it.blk_begin;
  const int lo = it.lo, hi = it.hi;

  // The lane's row: of the tile, of the request's (token, head) pairs.
  const int in_tile = wave * C::ROWS_WAVE + il;
  const int row = it.tile * C::ROWS_TILE + in_tile;
  const int token = row / p.group;
  u32x4 qf[C::KK];
  load_q<C>(p, it, row, in_tile < it.rows, hh, qf);
  const Seen seen = row_seen(p, it, token);
  // Blocks that end past the wave's first token's last key, or begin below its last token's first
  // key, hold keys that some row does not see.
  const int wave_row = it.tile * C::ROWS_TILE + wave * C::ROWS_WAVE;
  const int hi_min = row_seen(p, it, wave_row / p.group).hi;
  const int lo_max = row_seen(p, it, (wave_row + C::ROWS_WAVE - 1) / p.group).lo;

  float m = kNegBig, l = 0.0f;
  f32x16 o[C::DT];
#pragma unroll
  for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[dt][v] = 0.0f;

  // Each wave stages its output rows in its own part of the K ring (head-dim tile 64: of both
  // rings); the caller sees to it that nothing else uses that meanwhile.
  constexpr bool kStageInK = C::WAVES * 32 * kStagedRowBytes<C> <= C::NKSLOT * C::TILE_BYTES;
  auto store_output = [&]() {
    store_wave_rows<C>(p, it, wave * C::ROWS_WAVE, smem + wave * 32 * kStagedRowBytes<C>, lane, o, m, l);
  };
  if (N <= 0) {
    store_output();
    return;
  }

  const Lanes<C> ln(lane);
  const DmaLanes<C> dl(lane, wave, row_bytes);
  const BlockDma<C> bd(dl, wave, row_bytes);
  const RowDma<C> rd(dl, p.dim, wave, lane);
  BlockWindow win0{0, unit_window<C>(p, table_b, row_bytes, key0, N, lo, hi, 0, wave, lane)};
  BlockWindow win1{1, 0};
  // K and V of block j < N into slot j % 4 of the rings.
  auto issue_block = [&](int j, auto jslot) {
    if (j / C::WINDOW != win0.w) {
      win0 = win1;
      win1 = BlockWindow{win0.w + 1, unit_window<C>(p, table_b, row_bytes, key0, N, lo, hi, win0.w + 1, wave, lane)};
    }
    const u32 kdst = kring_lds + (u32)((int)jslot * C::TILE_BYTES);
    const u32 vdst = vring_lds + (u32)((int)jslot * C::TILE_BYTES);
    int pos0 = key0 + j * C::BN;
    asm volatile("" : "+s"(pos0));  // no induction variables for the rare path
    if constexpr (C::ROWS != kRowsBlock) {
#pragma unroll
      for (int q = 0; q < C::INSTR_PER_WAVE; ++q) {
        const int64_t off = readlane64(win0.off, j % C::WINDOW * C::INSTR_PER_WAVE + q);
        const u32 at = 1024u * (u32)(q * C::NWQ + wave);
        if ((int32_t)((uint64_t)off >> 32) >= 0) {
          issue_row_group<C>(kb + off, rd.k[q], rd.k_live[q], kdst + at);
          issue_row_group<C>(vb + off, rd.v[q], rd.v_live[q], vdst + at);
        } else {
          issue_keys<C, false>(p, table_b, kb, row_bytes, pos0, lo, hi, kdst, wave, lane, q);
          issue_keys<C, true>(p, table_b, vb, row_bytes, pos0, lo, hi, vdst, wave, lane, q);
        }
      }
    } else {
      const int64_t off = readlane64(win0.off, j % C::WINDOW);
      if ((int32_t)((uint64_t)off >> 32) >= 0) {
        issue_fast_block<C>(kb + off, vb + off, kdst, vdst, bd, wave);
      } else {
#pragma unroll
        for (int q = 0; q < C::INSTR_PER_WAVE; ++q) {
          issue_keys<C, false>(p, table_b, kb, row_bytes, pos0, lo, hi, kdst, wave, lane, q);
          issue_keys<C, true>(p, table_b, vb, row_bytes, pos0, lo, hi, vdst, wave, lane, q);
        }
      }
    }
  };
  // Block j has landed; the batch of block j + 1, issued after it, may be in flight.
  auto wait_block = [&](int j) {
    if (j + 1 < N)
      wait_vm<C::BATCH>();
    else
      wait_vm<0>();
  };
  constexpr std::integral_constant<int, 0> s0{};
  constexpr std::integral_constant<int, 1> s1{};
  constexpr std::integral_constant<int, 2> s2{};
  constexpr std::integral_constant<int, 3> s3{};
  issue_block(0, s0);
  if (1 < N) issue_block(1, s1);
  win1.off = unit_window<C>(p, table_b, row_bytes, key0, N, lo, hi, 1, wave, lane);
  wait_block(0);
  // (Q is older than block 0: the compiler's wait for it comes here, once, and not in the loop,
  // where it would cover the DMA in flight.)
#pragma unroll
  for (int kk = 0; kk < C::KK; ++kk) asm volatile("" ::"v"(qf[kk]));
  __syncthreads();

  f32x16 s[C::ST];
  u32x4 pf[C::KS];
  const OperandAddr<C> ad(ln, kring_lds, vring_lds);
  auto mphase = [&](auto slot, auto pv, auto qk) {
    const u32 ks = (u32)((int)slot * C::TILE_BYTES), vs = (u32)((((int)slot + 3) & 3) * C::TILE_BYTES);
    matrix_phase<C, decltype(pv)::value, decltype(qk)::value>(ad, ks, vs, qf, pf, s, o);
  };
  constexpr std::true_type on{};
  constexpr std::false_type off{};
  auto sphase = [&](int n) {
    int pos0 = key0 + n * C::BN;
    if (pos0 + C::BN > hi_min || pos0 < lo_max) {
      asm volatile("" : "+s"(pos0));
      mask_seen<C>(s, pos0, seen, hh);
    }
    online_softmax<C>(s, m, l, o, p.scale_log2, pf);
  };
  // The phases of prefill_kernel: group A runs M(n) in phase 2 n and S(n) in phase 2 n + 1, group B
  // one phase later; block n + 2 is issued in phase 2 n, and block n + 1 has landed at the end of
  // phase 2 n + 1. After the barrier that ends phase 2 N - 1 no DMA is in flight and nothing reads
  // the K ring, where the output rows are staged. Both groups pass the same barriers.
  if (opaque_uniform(wave) < C::WAVES / 2) {
    auto body = [&](int n, auto slot) {
      if (n + 2 < N) issue_block(n + 2, ((int)slot + 2) & 3);
      mphase(slot, on, on);
      __syncthreads();
      sphase(n);
      wait_block(n + 1);
      __syncthreads();
    };
    if (2 < N) issue_block(2, s2);
    mphase(s0, off, on);
    __syncthreads();
    sphase(0);
    wait_block(1);
    __syncthreads();
    int n = 1;
    for (; n + 4 <= N; n += 4) {
      body(n, s1);
      body(n + 1, s2);
      body(n + 2, s3);
      body(n + 3, s0);
    }
    for (; n < N; ++n) body(n, n & 3);
    mphase(N & 3, on, off);
    __syncthreads();
    if constexpr (!kStageInK) __syncthreads();  // group B no longer reads the V ring
    store_output();
  } else {
    auto body = [&](int n, auto slot) {
      if (n + 2 < N) issue_block(n + 2, ((int)slot + 2) & 3);
      sphase(n - 1);
      __syncthreads();
      mphase(slot, on, on);
      wait_block(n + 1);
      __syncthreads();
    };
    if (2 < N) issue_block(2, s2);
    __syncthreads();
    mphase(s0, off, on);
    wait_block(1);
    __syncthreads();
    int n = 1;
    for (; n + 4 <= N; n += 4) {
      body(n, s1);
      body(n + 1, s2);
      body(n + 2, s3);
      body(n + 3, s0);
    }
    for (; n < N; ++n) body(n, n & 3);
    sphase(N - 1);
    __syncthreads();
    mphase(N & 3, on, off);
    if constexpr (!kStageInK) __syncthreads();
    store_output();
  }
}

template <bool BF16, int DPAD, int ROWS>
hipError_t launch_extend_long(const ExtendParams& p, int grid, hipStream_t stream) {
  using C = PCfg<BF16, DPAD, ROWS>;
  extend_long_kernel<C><<<dim3(grid), dim3(C::THREADS), 0, stream>>>(p, p.table, p.lengths, p.cu);
  return hipGetLastError();
}

}  // namespace fgw_kv
