// Long tiles of the attention over pages (fgw_kv_extend) with head dims above 128: 128 rows of
// (token, head of the group), eight waves.
//
// The K/V ring of extend_long_kernel does not fit a CU's LDS at this head-dim tile, nor do its
// operands fit the registers; this is fwd_kernel's kDual arrangement (fmha_kernel.h): two sets of
// four waves hold the same 128 rows, each takes 32 keys of every 64-key block through two stages of
// its own, and their states meet in LDS at the end, so that one set's softmax runs beside the other's
// products (P rounded once, as in extend_long_kernel). Bound by the chain of a block (two waves to a
// SIMD at 256 registers). Hq 32, Hkv 8, 4096 tokens causal: D 256 424 us (649 TFLOP/s), D 192 433;
// 512 tokens behind 7680 cached ones, D 256, 210. The kernel of few rows takes 787, 841 and 327 for
// them.
#pragma once
#include "kv_extend_long.h"

namespace fgw_kv {

template <class C>
__global__ __launch_bounds__(C::THREADS) void extend_wide_kernel(ExtendParams p, const int32_t* __restrict__ table,
                                                                 const int32_t* __restrict__ lengths,
                                                                 const int32_t* __restrict__ cu) {
  static_assert(C::DUAL && C::NBUF == 2 && C::ROWS_TILE == WideTiling::ROWS && C::BLOCK == WideTiling::BN,
                "two sets of waves, two stages each");
  __shared__ __attribute__((aligned(1024))) unsigned char smem[C::LDS_BYTES];
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, il = lane & 31, hh = lane >> 5;
  const int wq = wave % C::NWQ, wk = wave / C::NWQ;
  Item it;
  const bool found = find_item<WideTiling>(p, lengths, cu, (int)blockIdx.x, lane, it);
  write_note(p, it, found);
  if (!found) return;

  const int N = it.blk_end - it.blk_begin;
  const int first_pos = it.blk_begin * C::BLOCK + wk * C::BN;
  KeyStream<C, false> keys(p, table, it, lane, wq, first_pos, C::BLOCK, N);
  const DmaLanes<C> dl(lane, wq, keys.row_bytes);
  const int in_tile = wq * C::ROWS_WAVE + il, row = it.tile * C::ROWS_TILE + in_tile;
  u32x4 qf[C::KK];
  load_q<C>(p, it, row, in_tile < it.rows, hh, qf);
  const Seen seen = row_seen(p, it, row / p.group);
  const int wave_row = it.tile * C::ROWS_TILE + wq * C::ROWS_WAVE;
  const int hi_min = row_seen(p, it, wave_row / p.group).hi;
  const int lo_max = row_seen(p, it, (wave_row + C::ROWS_WAVE - 1) / p.group).lo;

  const Lanes<C> ln(lane);
  unsigned char* const group = smem + wk * C::GROUP_BYTES;
  const u32 group_lds = lds_address(group);
  float m = kNegBig, l = 0.0f;
  f32x16 o[C::DT];
#pragma unroll
  for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[dt][v] = 0.0f;
  auto issue = [&](int n) {
    const u32 dst = group_lds + (u32)(n % 2 * C::STAGE_BYTES);
    keys.template issue<false>(dl, n, dst);
    keys.template issue<true>(dl, n, dst + (u32)C::TILE_BYTES);
  };
  keys.ids_ready();
  if (N > 0) issue(0);
#pragma unroll
  for (int kk = 0; kk < C::KK; ++kk) asm volatile("" ::"v"(qf[kk]));
  for (int n = 0; n < N; ++n) {
    const int pos0 = first_pos + C::BLOCK * n;
    const unsigned char* stage = group + n % 2 * C::STAGE_BYTES;
    wait_vm<0>();
    __syncthreads();  // tile n is in LDS; every wave is done with tile n - 1
    if (n + 1 < N) issue(n + 1);
    f32x16 s[C::ST];
    u32x4 pf[C::KS];
    qk_block<C>(stage, ln, qf, s);
    if (pos0 + C::BN > hi_min || pos0 < lo_max) mask_seen<C>(s, pos0, seen, hh);
    online_softmax<C>(s, m, l, o, p.scale_log2, pf);
    pv_block<C>(stage + C::TILE_BYTES, ln, pf, o);
  }
  // The second set's state to the first through LDS, lane to lane.
  __syncthreads();
  f32x4* const so = reinterpret_cast<f32x4*>(smem + wq * C::DT * 4096);
  float* const sml = reinterpret_cast<float*>(smem + C::NWQ * C::DT * 4096 + wq * 512);
  const int lo = opaque_lane(lane);
  if (wk == 1) {
    sml[lo] = m;
    sml[64 + lo] = l;
#pragma unroll
    for (int i = 0; i < 4 * C::DT; ++i)
      so[i * 64 + lo] = f32x4{o[i / 4][4 * (i % 4)], o[i / 4][4 * (i % 4) + 1], o[i / 4][4 * (i % 4) + 2],
                              o[i / 4][4 * (i % 4) + 3]};
  }
  __syncthreads();
  if (wk == 0) {
    const float mb = sml[lo], top = fmaxf(m, mb);
    const float wa = __builtin_amdgcn_exp2f(m - top), wb = __builtin_amdgcn_exp2f(mb - top);
    l = l * wa + sml[64 + lo] * wb;
    m = top;
#pragma unroll
    for (int i = 0; i < 4 * C::DT; ++i) {
      const f32x4 x = so[i * 64 + lo];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i / 4][4 * (i % 4) + j] = o[i / 4][4 * (i % 4) + j] * wa + x[j] * wb;
    }
  }
  __syncthreads();  // the states are read: the rows are staged there
  if (wk == 0)
    store_wave_rows<C>(p, it, wq * C::ROWS_WAVE, smem + wq * 32 * kStagedRowBytes<C>, lane, o, m, l);
}

template <bool BF16>
hipError_t launch_extend_wide(const ExtendParams& p, int grid, hipStream_t stream) {
  using C = Cfg<BF16, 256, kLayoutQuery, 0, kDual>;
  extend_wide_kernel<C><<<dim3(grid), dim3(C::THREADS), 0, stream>>>(p, p.table, p.lengths, p.cu);
  return hipGetLastError();
}

}  // namespace fgw_kv
