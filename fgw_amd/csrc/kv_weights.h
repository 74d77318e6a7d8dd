// Attention weight of cached keys (fgw_kv_weights): for each request, K/V head and key j,
//
//   scores[j] = (j < len - n ? decay scores[j] : 0) + sum over rows R of exp2(s_Rj - L_R),
//
// where the rows are the (token, head of the group) pairs of the request's last min(n, last) new tokens,
// s_Rj = q_R . k_j scale log2(e) for the keys up to the row's own token, and L_R = log2 sum_j exp2(s_Rj).
// L_R needs all keys of a row before the first weight is known, and keys come in splits, so there are
// two passes. Scores, statistics and sums are fp32; no sum's order hangs on the order of programs.
//
// Few rows (up to kKeptRows of a request and K/V head: a decode step). Memory bounds it, so K is read once:
//   weights_rows_kernel    s = Q K^T as the kernel of few rows of fgw_kv_extend has it (four waves, each
//                          with 32-key tiles of its own on the way through LDS), kept in the workspace;
//                          the split's L. A tile of one split is finished at once.
//   weights_finish_kernel  L of the row from its splits', and the kept scores' exponentials.
// More rows. K is read twice, which costs little beside the products:
//   weights_stats_kernel   L: tiles of 128 rows, four waves with 32 rows each, all keys past them;
//   weights_columns_kernel the other way round: four waves hold 32 keys each, and up to kColumnRows rows of
//                          Q go past them, so a lane adds up its own key's weights;
//   weights_sum_kernel     where a request has more rows than that: the parts' sums.
#pragma once
#include "kv_extend.h"

namespace fgw_kv {

constexpr int kKeptRows = 16;
constexpr int kColumnRows = 1024;  // rows of a part
constexpr int kColumnKeys = 128;   // keys of an item
constexpr int kSumKeys = 1024;

struct WeightParams : ExtendParams {
  float* scores;    // [batch, heads, stride]
  int64_t stride;
  float* kept;      // few rows: [batch, heads, kept_rows, keys_pad] scores in log2 units
  float* sums;      // more rows: [parts, heads, keys_pad]
  int32_t* request_notes;  // more rows: [batch] WeightNote
  int32_t last, kept_rows, keys_pad, parts_most;
  float decay;
};
template <>
inline constexpr bool kPicksFrom<WeightParams> = true;

// Where the statistics of a request's tiles are: those of its first item (a place for each K/V head), the
// splits of its tiles at most, how many tiles, and the units of a split.
struct WeightNote {
  int32_t base, splits, tiles, chunk;
};

typedef Tiling<128, 64, 1> StatsTiling;

// The request's last tokens alone are its rows; `from` says where its new keys begin.
template <class T>
__device__ __forceinline__ Request load_request(const WeightParams& p, const int32_t* lengths, const int32_t* cu, int b) {
  Request r{0, 0, 0, 0, 0, 0, 0, -1};
  if (b >= p.batch) return r;
  const int first = cu[b], next = cu[b + 1], capacity = p.width * p.page_size;
  int len = lengths[b];
  len = len < 0 ? 0 : (len > capacity ? capacity : len);
  if (first < 0 || next > p.tokens || next <= first || len == 0) return r;
  const int n = next - first;
  r.n = n < p.last ? n : p.last;
  r.first = next - r.n;
  r.len = len;
  r.from = len > n ? len - n : 0;
  r.tiles = (int)(((int64_t)r.n * p.group + T::ROWS - 1) / T::ROWS);
  r.units = (len + T::KEYS - 1) / T::KEYS;
  return r;
}

__device__ __forceinline__ float lse2_of(float m, float total) {
  return total > 0.0f ? m + __builtin_amdgcn_logf(total) : total == total ? kNegBig : total;
}

// sum exp2 of s scale - m over a lane's scores, without the packing of softmax_exp.
__device__ __forceinline__ float exp_sum(const f32x16& s, float m, float scale_log2) {
  float rs[4];
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[v], scale_log2, -m));
    rs[v % 4] = v < 4 ? e : rs[v % 4] + e;
  }
  return (rs[0] + rs[1]) + (rs[2] + rs[3]);
}

// A key's running sum: keys that the new tokens brought begin anew.
__device__ __forceinline__ void add_score(const WeightParams& p, float* row, int key, int from, float sum) {
  float old = 0.0f;
  if (key < from && p.decay != 0.0f) old = row[key] * p.decay;
  row[key] = old + sum;
}

// ---- few rows -----------------------------------------------------------------------------------

template <int DPAD>
constexpr int kWeightStages = DPAD >= 128 ? 2 : 4;

// Keys [from, to) of an item's tile: the kept scores of its rows against their L.
__device__ __forceinline__ void finish_keys(const WeightParams& p, const Item& it, const float* lse2, int from, int to,
                                            int tid, int threads) {
  const int64_t place = (int64_t)it.b * p.heads + it.head;
  const float* const kept = p.kept + place * p.kept_rows * p.keys_pad;
  float* const row = p.scores + place * p.stride;
  for (int key = from + tid; key < to; key += threads) {
    float sum = 0.0f;
    for (int r = 0; r < it.rows; ++r) {
      const float s = kept[(int64_t)r * p.keys_pad + key];
      sum += s == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s - lse2[r]);
    }
    add_score(p, row, key, it.from, sum);
  }
}

template <class C>
__global__ __launch_bounds__(C::THREADS, C::DPAD == 256 ? 1 : 2) void weights_rows_kernel(
    WeightParams p, const int32_t* __restrict__ table, const int32_t* __restrict__ lengths, const int32_t* __restrict__ cu) {
  constexpr int S = kWeightStages<C::DPAD>;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[C::NWK * S * C::TILE_BYTES];
  __shared__ float cm[C::NWK * kKeptRows], cl[C::NWK * kKeptRows], clse[kKeptRows];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int il = lane & 31, hh = lane >> 5;
  Item it;
  if (!find_item<ShortTiling>(p, lengths, cu, (int)blockIdx.x, lane, it)) return;
  const Lanes<C> ln(lane);
  unsigned char* const stages = smem + wave * S * C::TILE_BYTES;
  const u32 stages_lds = lds_address(stages);

  constexpr int kStep = C::NWK * C::BN;
  const int cnt = it.blk_end - it.blk_begin;
  const int my_n = cnt > wave ? (cnt - wave + C::NWK - 1) / C::NWK : 0;
  const int first_pos = (it.blk_begin + wave) * C::BN;
  KeyStream<C> keys(p, table, it, lane, 0, first_pos, kStep, my_n);
  const DmaLanes<C> dl(lane, 0, keys.row_bytes);
  auto issue = [&](int n) { keys.template issue<false>(dl, n, stages_lds + (u32)(n % S * C::TILE_BYTES)); };

  u32x4 qf[C::KK];
  load_q<C>(p, it, il, il < it.rows, hh, qf);
  const Seen seen = row_seen(p, it, il / p.group);
  const int hi_min = row_seen(p, it, 0).hi;
  float* const kept = p.kept + (((int64_t)it.b * p.heads + it.head) * p.kept_rows + il) * p.keys_pad;

  float m = kNegBig, l = 0.0f;
  keys.ids_ready();
  for (int n = 0; n < S && n < my_n; ++n) issue(n);
#pragma unroll
  for (int kk = 0; kk < C::KK; ++kk) asm volatile("" ::"v"(qf[kk]));
  for (int n = 0; n < my_n; ++n) {
    const int pos0 = first_pos + kStep * n, rem = my_n - 1 - n;
    const unsigned char* stage = stages + n % S * C::TILE_BYTES;
    // (Stores of kept scores may be in flight behind the tile too: that only makes the wait stricter.)
    if (rem >= S - 1)
      wait_vm<(S - 1) * C::INSTR>();
    else if (S > 2 && rem == 2)
      wait_vm<(S > 2 ? 2 : 0) * C::INSTR>();
    else if (S > 2 && rem == 1)
      wait_vm<(S > 2 ? 1 : 0) * C::INSTR>();
    else
      wait_vm<0>();
    asm volatile("" ::: "memory");
    u32x4 ka[C::KK];
#pragma unroll
    for (int kk = 0; kk < C::KK; ++kk) ka[kk] = read_k<C>(stage, ln, 0, kk);
    wait_lds();
    __builtin_amdgcn_sched_barrier(0);
    if (rem >= S) issue(n + S);
    f32x16 s[1], t;
#pragma unroll
    for (int v = 0; v < 16; ++v) s[0][v] = t[v] = 0.0f;
#pragma unroll
    for (int kk = 0; kk < C::KK; kk += 2) {
      s[0] = Elem<C::BF16>::mma(ka[kk], qf[kk], s[0]);
      t = Elem<C::BF16>::mma(ka[kk + 1], qf[kk + 1], t);
    }
    s[0] += t;
    if (pos0 + C::BN > hi_min) mask_seen<C>(s, pos0, seen, hh);
    float sum = exp_sum(s[0], m, p.scale_log2);
    if (__ballot(!(sum <= kSoftmaxSumBound))) {
      const float top = fmaxf(m, row_max<C>(s, p.scale_log2));
      l *= __builtin_amdgcn_exp2f(m - top);
      m = top;
      sum = exp_sum(s[0], m, p.scale_log2);
    }
    l += sum;
    if (il < it.rows) {
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(kept + pos0 + 8 * g + 4 * hh) =
            f32x4{s[0][4 * g], s[0][4 * g + 1], s[0][4 * g + 2], s[0][4 * g + 3]} * p.scale_log2;
    }
  }

  const float tot = pair_sum(l);
  if (hh == 0 && il < it.rows) {
    cm[wave * kKeptRows + il] = m;
    cl[wave * kKeptRows + il] = tot;
  }
  wait_vm<0>();  // the kept scores of every wave
  __syncthreads();
  if (tid < it.rows) {
    float mm = kNegBig, t2 = 0.0f;
#pragma unroll
    for (int k = 0; k < C::NWK; ++k) mm = fmaxf(mm, cm[k * kKeptRows + tid]);
#pragma unroll
    for (int k = 0; k < C::NWK; ++k) t2 += cl[k * kKeptRows + tid] * __builtin_amdgcn_exp2f(cm[k * kKeptRows + tid] - mm);
    const float lse = lse2_of(mm, t2);
    clse[tid] = lse;
    if (it.splits > 1) p.lse[(int64_t)it.slot * kKeptRows + tid] = lse;
  }
  if (it.splits > 1) return;
  __syncthreads();
  finish_keys(p, it, clse, 0, it.len, tid, C::THREADS);
}

// The items of weights_rows_kernel again, those of split tiles.
constexpr int kFinishThreads = 256;
static __global__ __launch_bounds__(kFinishThreads) void weights_finish_kernel(WeightParams p,
                                                                              const int32_t* __restrict__ lengths,
                                                                              const int32_t* __restrict__ cu) {
  __shared__ float part[kFinishThreads], clse[kKeptRows];
  const int tid = threadIdx.x;
  Item it;
  if (!find_item<ShortTiling>(p, lengths, cu, (int)blockIdx.x, tid & 63, it) || it.splits == 1) return;
  // 16 threads to a row, then its first one.
  const int r = tid % kKeptRows, g = tid / kKeptRows;
  constexpr int kShare = kFinishThreads / kKeptRows;
  float m = kNegBig, l = 0.0f;
  if (r < it.rows) {
    for (int s = g; s < it.splits; s += kShare) {
      const float x = p.lse[(int64_t)(it.slot0 + s * it.slot_step) * kKeptRows + r], top = fmaxf(m, x);
      l = l * __builtin_amdgcn_exp2f(m - top) + __builtin_amdgcn_exp2f(x - top);
      m = top;
    }
  }
  part[tid] = l > 0.0f || l != l ? lse2_of(m, l) : kNegBig;
  __syncthreads();
  if (tid < it.rows) {
    float top = kNegBig, sum = 0.0f;
    for (int k = 0; k < kShare; ++k) top = fmaxf(top, part[k * kKeptRows + tid]);
    for (int k = 0; k < kShare; ++k) sum += __builtin_amdgcn_exp2f(part[k * kKeptRows + tid] - top);
    clse[tid] = lse2_of(top, sum);
  }
  __syncthreads();
  const int from = it.blk_begin * ShortTiling::BN, to = it.blk_end * ShortTiling::BN;
  finish_keys(p, it, clse, from, to < it.len ? to : it.len, tid, kFinishThreads);
}

// ---- more rows ----------------------------------------------------------------------------------

// Four waves that share 32-row tiles of K or Q in LDS, two tiles to a step.
template <bool BF16_, int DPAD_>
struct WCfg {
  static constexpr bool BF16 = BF16_;
  static constexpr int DPAD = DPAD_, NWQ = 4, NWK = 1, BN = 32, THREADS = 256, ROWS_WAVE = 32, ROWS_TILE = 128;
  static constexpr int KK = DPAD / 16, ST = 1, KS = 2, CPR = DPAD / 8, ROW_BYTES = DPAD * 2;
  static constexpr int TILE_BYTES = BN * ROW_BYTES, INSTR = TILE_BYTES / 1024, INSTR_PER_WAVE = INSTR / NWQ;
  static constexpr int KSW = CMin<16, CPR>::value, VSW = CPR / 4, RPI = 64 / CPR;
  static constexpr int STEP_BYTES = 2 * TILE_BYTES;
  static constexpr int STAGES = DPAD == 256 ? 2 : 3;
  static_assert(DPAD >= 64 && INSTR_PER_WAVE >= 1, "DMA granularity");
};

// The step loop of both kernels: step j's two tiles have landed for all waves when work(j, stage) runs.
template <class C, class Issue, class Work>
__device__ __forceinline__ void stream_steps(int steps, Issue&& issue, Work&& work) {
  constexpr int kAhead = C::STAGES - 1, kBatch = 2 * C::INSTR_PER_WAVE;
  for (int j = 0; j < kAhead && j < steps; ++j) issue(j, j);
  int stage = 0;
  for (int j = 0; j < steps; ++j) {
    if (kAhead > 1 && j + 1 < steps)
      wait_vm<(kAhead - 1) * kBatch>();
    else
      wait_vm<0>();
    __syncthreads();
    if (j + kAhead < steps) issue(j + kAhead, stage == 0 ? C::STAGES - 1 : stage - 1);
    work(j, stage);
    stage = stage + 1 == C::STAGES ? 0 : stage + 1;
  }
}

template <class C>
__global__ __launch_bounds__(C::THREADS, C::DPAD == 256 ? 2 : 3) void weights_stats_kernel(
    WeightParams p, const int32_t* __restrict__ table, const int32_t* __restrict__ lengths, const int32_t* __restrict__ cu) {
  __shared__ __attribute__((aligned(1024))) unsigned char smem[C::STAGES * C::STEP_BYTES];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int il = lane & 31, hh = lane >> 5;
  Item it;
  int chunk;
  if (!find_item<StatsTiling>(p, lengths, cu, (int)blockIdx.x, lane, it, &chunk)) return;
  if (it.place == 0 && it.head == 0 && tid == 0)
    reinterpret_cast<WeightNote*>(p.request_notes)[it.b] = WeightNote{(int)blockIdx.x / p.heads, it.place_splits, it.tiles, chunk};
  const int first_pos = it.blk_begin * StatsTiling::BN, tiles = 2 * (it.blk_end - it.blk_begin);
  KeyStream<C, false> keys(p, table, it, lane, wave, first_pos, C::BN, tiles);
  const DmaLanes<C> dl(lane, wave, keys.row_bytes);
  const u32 lds = lds_address(smem);
  const int in_tile = wave * C::ROWS_WAVE + il, row = it.tile * C::ROWS_TILE + in_tile;
  u32x4 qf[C::KK];
  load_q<C>(p, it, row, in_tile < it.rows, hh, qf);
  const Seen seen = row_seen(p, it, row / p.group);
  const int hi_min = row_seen(p, it, (it.tile * C::ROWS_TILE + wave * C::ROWS_WAVE) / p.group).hi;
  const Lanes<C> ln(lane);
  float m = kNegBig, l = 0.0f;
  keys.ids_ready();
#pragma unroll
  for (int kk = 0; kk < C::KK; ++kk) asm volatile("" ::"v"(qf[kk]));
  stream_steps<C>(
      tiles / 2,
      [&](int j, int stage) {
        keys.template issue<false>(dl, 2 * j, lds + (u32)(stage * C::STEP_BYTES));
        keys.template issue<false>(dl, 2 * j + 1, lds + (u32)(stage * C::STEP_BYTES + C::TILE_BYTES));
      },
      [&](int j, int stage) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int pos0 = first_pos + 64 * j + 32 * h;
          f32x16 s[1];
          qk_block<C>(smem + stage * C::STEP_BYTES + h * C::TILE_BYTES, ln, qf, s);
          if (pos0 + C::BN > hi_min) mask_seen<C>(s, pos0, seen, hh);
          float sum = exp_sum(s[0], m, p.scale_log2);
          if (__ballot(!(sum <= kSoftmaxSumBound))) {
            const float top = fmaxf(m, row_max<C>(s, p.scale_log2));
            l *= __builtin_amdgcn_exp2f(m - top);
            m = top;
            sum = exp_sum(s[0], m, p.scale_log2);
          }
          l += sum;
        }
      });
  const float tot = pair_sum(l);
  if (hh == 0 && in_tile < it.rows) p.lse[(int64_t)it.slot * C::ROWS_TILE + in_tile] = lse2_of(m, tot);
}

// Items of the other two kernels: key blocks times parts of the rows of each request and head, and
// blocks of keys of the requests with several parts.
struct Column {
  int b, head, first, n, len, from, block, part, parts, part0;
};
template <bool SUM>
__device__ __forceinline__ bool find_column(const WeightParams& p, const int32_t* lengths, const int32_t* cu, int64_t w,
                                            int lane, const Request& r0, Column& it) {
  const int64_t g64 = w / p.heads;
  it.head = (int)(w - g64 * p.heads);
  int64_t before = 0;
  int parts_before = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 64) {
    const Request r = b0 == 0 ? r0 : load_request<StatsTiling>(p, lengths, cu, b0 + lane);
    const int parts = r.tiles ? (int)(((int64_t)r.n * p.group + kColumnRows - 1) / kColumnRows) : 0;
    const int per = SUM ? (parts > 1 ? 1 : 0) : parts, keys = SUM ? kSumKeys : kColumnKeys;
    const int items = r.tiles ? (r.len + keys - 1) / keys * per : 0;
    const int items_to = wave_incl_sum(items, lane), parts_to = wave_incl_sum(parts, lane);
    const int64_t at = g64 - before - (items_to - items);
    const uint64_t hit = __ballot(at >= 0 && at < items);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      auto pick = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
      it.b = b0 + l;
      it.first = pick(r.first);
      it.n = pick(r.n);
      it.len = pick(r.len);
      it.from = pick(r.from);
      it.parts = pick(parts);
      it.part0 = parts_before + pick(parts_to - parts);
      const int place = pick((int)at), step = SUM ? 1 : it.parts;
      it.block = (int)((u32)place / (u32)step);
      it.part = place - it.block * step;
      return true;
    }
    before += __builtin_amdgcn_readlane(items_to, 63);
    parts_before += __builtin_amdgcn_readlane(parts_to, 63);
  }
  return false;
}
// The first row of a request that sees the key (rows see their token's own position and all before it).
__device__ __forceinline__ int first_row(const WeightParams& p, const Column& it, int key) {
  const int token = key - (it.len - it.n);
  return token > 0 ? token * p.group : 0;
}

template <class C>
__global__ __launch_bounds__(C::THREADS, C::DPAD == 256 ? 2 : 3) void weights_columns_kernel(
    WeightParams p, const int32_t* __restrict__ table, const int32_t* __restrict__ lengths, const int32_t* __restrict__ cu) {
  __shared__ __attribute__((aligned(1024))) unsigned char smem[C::STAGES * C::STEP_BYTES];
  __shared__ __attribute__((aligned(16))) float slse[kColumnRows + 64];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int il = lane & 31, hh = lane >> 5;
  const u32 lds = lds_address(smem);
  const Lanes<C> ln(lane);
  const Request r0 = load_request<StatsTiling>(p, lengths, cu, lane);
  const int64_t row_bytes = (int64_t)p.heads * p.dim * 2;
  Column it;
  for (int64_t w = blockIdx.x; find_column<false>(p, lengths, cu, w, lane, r0, it); w += gridDim.x) {
    const int rows = it.n * p.group, key0 = it.block * kColumnKeys;
    const int end = rows - it.part * kColumnRows < kColumnRows ? rows : (it.part + 1) * kColumnRows;
    // (Steps of 64 rows from the part's first row.)
    const int part0 = it.part * kColumnRows, seen0 = first_row(p, it, key0);
    if (seen0 >= end) continue;
    const int begin = seen0 > part0 ? part0 + (seen0 - part0) / 64 * 64 : part0, steps = (end - begin + 63) / 64;

    // K of the lane's key, from its page.
    const int key = key0 + wave * 32 + il;
    const u32 pg = key < it.len ? div_page((u32)key, p.page_magic, p.page_shift) : 0u;
    const int64_t krow = (int64_t)table[(int64_t)it.b * p.width + pg] * p.page_size + ((u32)key - pg * (u32)p.page_size);
    const bool live = key < it.len && krow >= 0 && krow < p.pool_rows;
    const char* const kp = static_cast<const char*>(p.k) + (int64_t)it.head * p.dim * 2 + (live ? krow * row_bytes : 0);
    u32x4 kf[C::KK];
#pragma unroll
    for (int kk = 0; kk < C::KK; ++kk) {
      const int d = 16 * kk + 8 * hh;
      u32x4 x = {0u, 0u, 0u, 0u};
      if (live && d < p.dim) x = *reinterpret_cast<const u32x4*>(kp + 2 * d);
      kf[kk] = x;
    }
    // L of the part's rows, from their splits.
    __syncthreads();  // the item before is done with slse and the stages
    const WeightNote note = reinterpret_cast<const WeightNote*>(p.request_notes)[it.b];
    for (int r = begin + tid; r < begin + 64 * steps; r += C::THREADS) {
      float lse = INFINITY;  // rows that are none weigh nothing
      if (r < end) {
        const int tile = r / C::ROWS_TILE, last = (tile + 1) * C::ROWS_TILE < rows ? (tile + 1) * C::ROWS_TILE : rows;
        int hi = it.len - it.n + (last - 1) / p.group + 1;
        hi = hi < 0 ? 0 : hi;
        const int most = splits_of(p, (hi + StatsTiling::KEYS - 1) / StatsTiling::KEYS, note.chunk);
        const int splits = most < note.splits ? most : note.splits;
        const int64_t slot = (int64_t)(note.base + (note.tiles - 1 - tile) * note.splits) * p.heads + it.head;
        float m = kNegBig, l = 0.0f;
        for (int s = 0; s < splits && slot + (int64_t)s * p.heads < p.work && slot >= 0; ++s) {
          const float x = p.lse[(slot + (int64_t)s * p.heads) * C::ROWS_TILE + (r - tile * C::ROWS_TILE)], top = fmaxf(m, x);
          l = l * __builtin_amdgcn_exp2f(m - top) + __builtin_amdgcn_exp2f(x - top);
          m = top;
        }
        lse = m > 0.5f * kNegBig || l != l ? lse2_of(m, l) : INFINITY;
      }
      slse[r - begin] = lse;
    }
#pragma unroll
    for (int kk = 0; kk < C::KK; ++kk) asm volatile("" ::"v"(kf[kk]));
    __syncthreads();

    // 32 rows of Q into LDS, a K tile's layout.
    auto issue_tile = [&](int row0, u32 dst) {
      const char* zero = reinterpret_cast<const char*>(kZeroChunk);
      const int at = lane % C::CPR;
#pragma unroll
      for (int q = 0; q < C::INSTR_PER_WAVE; ++q) {
        const int i = q * C::NWQ + wave, r = C::RPI * i + lane / C::CPR, row = row0 + r, c = at ^ (r % C::KSW);
        const int token = (int)((u32)row / (u32)p.group), head = row - token * p.group;
        const char* src = static_cast<const char*>(p.q) + (int64_t)(it.first + token) * p.q_token +
                          (int64_t)(it.head * p.group + head) * p.q_head + c * 16;
        dma_flat(row < end && c * 8 < p.dim ? src : zero, dst + 1024u * (u32)i);
      }
    };
    const int mine = first_row(p, it, key), all = first_row(p, it, key0 + wave * 32 + 31);
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    stream_steps<C>(
        steps,
        [&](int j, int stage) {
          issue_tile(begin + 64 * j, lds + (u32)(stage * C::STEP_BYTES));
          issue_tile(begin + 64 * j + 32, lds + (u32)(stage * C::STEP_BYTES + C::TILE_BYTES));
        },
        [&](int j, int stage) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int at = 64 * j + 32 * h;
            f32x16 s[1];
            qk_block<C>(smem + stage * C::STEP_BYTES + h * C::TILE_BYTES, ln, kf, s);
            f32x4 lse[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) lse[g] = *reinterpret_cast<const f32x4*>(slse + at + 8 * g + 4 * hh);
            if (begin + at >= all) {
#pragma unroll
              for (int v = 0; v < 16; ++v)
                acc[v % 4] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][v], p.scale_log2, -lse[v / 4][v % 4]));
            } else {
#pragma unroll
              for (int v = 0; v < 16; ++v) {
                const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][v], p.scale_log2, -lse[v / 4][v % 4]));
                acc[v % 4] += begin + at + 8 * (v / 4) + 4 * hh + v % 4 >= mine ? e : 0.0f;
              }
            }
          }
        });
    const float sum = pair_sum((acc[0] + acc[1]) + (acc[2] + acc[3]));
    if (hh == 0 && key < it.len) {
      if (it.parts == 1)
        add_score(p, p.scores + ((int64_t)it.b * p.heads + it.head) * p.stride, key, it.from, sum);
      else if (it.part0 + it.part < p.parts_most)
        p.sums[((int64_t)(it.part0 + it.part) * p.heads + it.head) * p.keys_pad + key] = sum;
    }
  }
}

static __global__ __launch_bounds__(kFinishThreads) void weights_sum_kernel(WeightParams p, const int32_t* __restrict__ lengths,
                                                                           const int32_t* __restrict__ cu) {
  const int tid = threadIdx.x, lane = tid & 63;
  const Request r0 = load_request<StatsTiling>(p, lengths, cu, lane);
  Column it;
  for (int64_t w = blockIdx.x; find_column<true>(p, lengths, cu, w, lane, r0, it); w += gridDim.x) {
    const int end = it.len < (it.block + 1) * kSumKeys ? it.len : (it.block + 1) * kSumKeys;
    float* const row = p.scores + ((int64_t)it.b * p.heads + it.head) * p.stride;
    for (int key = it.block * kSumKeys + tid; key < end; key += kFinishThreads) {
      // Parts whose rows all come before the key's block left nothing.
      float sum = 0.0f;
      for (int c = first_row(p, it, key / kColumnKeys * kColumnKeys) / kColumnRows; c < it.parts; ++c)
        if (it.part0 + c < p.parts_most) sum += p.sums[((int64_t)(it.part0 + c) * p.heads + it.head) * p.keys_pad + key];
      add_score(p, row, key, it.from, sum);
    }
  }
}

template <bool BF16, int DPAD>
hipError_t launch_weights(const WeightParams& p, bool many, int grid, int columns, hipStream_t stream) {
  if (!many) {
    using C = Cfg<BF16, DPAD, kLayoutKey, DPAD == 128 ? 1 : 0>;
    weights_rows_kernel<C><<<dim3(grid), dim3(C::THREADS), 0, stream>>>(p, p.table, p.lengths, p.cu);
  } else {
    using C = WCfg<BF16, DPAD>;
    weights_stats_kernel<C><<<dim3(grid), dim3(C::THREADS), 0, stream>>>(p, p.table, p.lengths, p.cu);
    weights_columns_kernel<C><<<dim3(columns), dim3(C::THREADS), 0, stream>>>(p, p.table, p.lengths, p.cu);
  }
  return hipGetLastError();
}

}  // namespace fgw_kv
