// Attention weight of cached keys (fgw_kv_weights): for each request, K/V head and key j,
//
//   scores[j] = (j < len - n ? decay scores[j] : 0) + sum over rows R of exp2(s_Rj - L_R),
//
// where the rows are the (token, head of the group) pairs of the request's last min(n, last) new tokens,
// s_Rj = q_R . k_j scale log2(e) for the keys up to the row's own token, and L_R = log2 sum_j exp2(s_Rj).
// L_R needs all keys of a row before the first weight is known, and keys come in splits, so there are
// two passes. Scores, statistics and sums are fp32; no sum's order hangs on the order of programs.
//
// Few rows (up to kKeptRows of a request and K/V head: decode, draft tokens). Memory bounds it, so K is read once:
//   weights_rows_kernel    s = Q K^T as the kernel of few rows of fgw_kv_extend has it (four waves, each
//                          with 32-key tiles of its own on the way through LDS), kept in the workspace;
//                          the split's L. A tile of one split is finished at once.
//   weights_finish_kernel  L of the row from its splits', and the kept scores' exponentials.
// More rows. K is read twice, which costs little beside the products:
//   weights_stats_kernel   L: tiles of 256 rows, four waves with 64 rows each, all keys past them;
//   weights_columns_kernel the other way round: four waves hold 64 keys each, and up to kColumnRows rows of
//                          Q go past them, so a lane adds up its own key's weights;
//   weights_sum_kernel     where a request has more rows than that: the parts' sums.
// The last two go over a range of keys at a time, where the partial sums of all of them would be too many
// (kv_weights.hip).
//
// Measured (BF16, 8 K/V heads of 4 rows a token, D 128): one new token of each of 32 requests of up to 4096 keys 45
// us without the copy of the sums, 3.9 TB/s of K, bound by the longest item's reads (38 us; then 7 for the splits);
// two prompts of 4096 tokens 359 us, 383 TFLOP/s of the products that the weights need and twice that of those
// done (stats 191, columns 218 when profiled), bound by exponentials and products in turn: two for a visible pair
// of either kind, and masked halves of the diagonal's tiles. The last 32 tokens of three prompts of up to 12288
// keys (FP16, D 96): 34 us, two kernels of one wave of programs, 17 each, most of it their starts and ends.
#pragma once
#include "kv_extend.h"

#include "fmha_prefill.h"

namespace fgw_kv {

// Rows of a request and K/V head whose scores are kept, in tiles of 32 or 64. The more they are, the more the kept
// scores weigh against a second reading of K. Two passes over K / one with the scores kept, us, requests of 4096
// keys, 8 K/V heads: 20 rows, 32 of them 165 / 89, 36 rows 168 / 120, 48 rows 170 / 134, 64 rows 165 / 164 (8
// requests 50.8 / 49.5, one of 32768 keys 53 / 56); D 64, 16 requests, 20 rows 63 / 41, 48 rows 64 / 58; D 256, 36
// rows of 4 heads 98 / 62, 64 rows of 8 182 / 118.
constexpr int kKeptRows = 48, kKeptRowsWide = 64;  // (D > 128)
template <int NR>
using KeptTiling = Tiling<32 * NR, ShortTiling::BN, ShortTiling::UNIT>;
constexpr int kColumnRows = 1024;  // rows of a part at most
constexpr int kColumnKeys = 256;   // keys of an item, of its sums too
constexpr int kWaveSimd = 2;       // waves to a SIMD

struct WeightParams : ExtendParams {
  float* scores;    // [batch, heads, stride]
  int64_t stride;
  float* kept;      // few rows: [batch, heads, kept_rows, keys_pad] scores in log2 units
  float* sums;      // more rows: [parts, heads, keys_pad], of the keys of a launch
  int32_t* request_notes;  // more rows: [batch] WeightNote
  int32_t last, kept_rows, keys_pad, parts_most;
  int32_t part_rows, part_shift;  // rows of a part: kColumnRows or a half or a quarter of it; their log2
  int32_t block_from, block_to;   // blocks of kColumnKeys keys of a launch
  float decay;
};
template <>
inline constexpr bool kPicksFrom<WeightParams> = true;

// Where the statistics of a request's tiles are: those of its first item (a place for each K/V head), the
// splits of its tiles at most, how many tiles, and the units of a split.
struct WeightNote {
  int32_t base, splits, tiles, chunk;
};

typedef Tiling<256, 64, 1> StatsTiling;

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

// Tiles of a wave on the way. One leaves room for three programs on a CU; one / two, us: 256 requests of up to
// 512 keys 61 / 70, 32 of 4096 D 256 112 / 120, one of 32768 22.7 / 23.6.
template <int DPAD>
constexpr int kWeightStages = DPAD >= 128 ? 1 : 2;

// Keys [from, to) of an item's tile, from a multiple of 4: the kept scores of its rows against their L, four
// keys to a thread and four rows on the way at a time.
__device__ __forceinline__ void finish_keys(const WeightParams& p, const Item& it, const float* lse2, int from, int to,
                                            int tid, int threads) {
  const int64_t place = (int64_t)it.b * p.heads + it.head;
  const float* const kept = p.kept + place * p.kept_rows * p.keys_pad;
  float* const row = p.scores + place * p.stride;
  for (int key = from + 4 * tid; key < to; key += 4 * threads) {
    float old[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) old[i] = p.decay != 0.0f && key + i < to && key + i < it.from ? row[key + i] : 0.0f;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int r0 = 0; r0 < it.rows; r0 += 4) {
      f32x4 s[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)  // (the last row again where there are fewer: not added)
        s[k] = *reinterpret_cast<const f32x4*>(kept + (int64_t)(r0 + k < it.rows ? r0 + k : it.rows - 1) * p.keys_pad + key);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float lse = lse2[r0 + k < it.rows ? r0 + k : 0];
        // Keys that the row sees: its own are NaN where L is, also one whose score is minus infinity, as those
        // that it does not see are kept. (Those weigh nothing beside any other L.)
        int hi = r0 + k < it.rows ? to : 0;
        if (lse != lse && r0 + k < it.rows) hi = row_seen(p, it, (r0 + k) / p.group).hi;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] += key + i < hi ? __builtin_amdgcn_exp2f(s[k][i] - lse) : 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (key + i < to) row[key + i] = (p.decay != 0.0f ? old[i] * p.decay : 0.0f) + sum[i];
  }
}

// LDS writes and reads of one wave keep their order (the hardware does; this is for the compiler).
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

template <class C, int NR>
__global__ __launch_bounds__(C::THREADS, C::DPAD == 256 ? 1 : 2) void weights_rows_kernel(
    WeightParams p, const int32_t* __restrict__ table, const int32_t* __restrict__ lengths, const int32_t* __restrict__ cu) {
  constexpr int S = kWeightStages<C::DPAD>, ROWS = 32 * NR;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[C::NWK * S * C::TILE_BYTES];
  // The scores of a wave's last tile, row by row: written to the workspace from here a tile later, whole
  // rows of 128 bytes (straight from the lanes that hold them, 16 bytes each, the stores took a fifth of the
  // time: 32 requests of 4096 keys 78 us, without any of them 64).
  constexpr int kRow = 36;
  __shared__ __attribute__((aligned(16))) float out[C::NWK][ROWS * kRow];
  __shared__ float cm[C::NWK * ROWS], cl[C::NWK * ROWS], clse[ROWS];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int il = lane & 31, hh = lane >> 5;
  Item it;
  if (!find_item<KeptTiling<NR>>(p, lengths, cu, (int)blockIdx.x, lane, it)) return;
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

  u32x4 qf[NR][C::KK];
  Seen seen[NR];
  float m[NR], l[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int row = 32 * r + il;
    load_q<C>(p, it, row < it.rows ? row : 0, row < it.rows, hh, qf[r]);
    seen[r] = row_seen(p, it, row / p.group);
    m[r] = kNegBig;
    l[r] = 0.0f;
  }
  const int hi_min = row_seen(p, it, 0).hi;
  float* const kept = p.kept + ((int64_t)it.b * p.heads + it.head) * p.kept_rows * p.keys_pad;
  auto store_kept = [&](int pos0) {  // 8 rows at a time, 8 lanes to a row
    for (int r = lane / 8; r < it.rows; r += 8)
      *reinterpret_cast<f32x4*>(kept + (int64_t)r * p.keys_pad + pos0 + 4 * (lane % 8)) =
          *reinterpret_cast<const f32x4*>(&out[wave][r * kRow + 4 * (lane % 8)]);
  };

  keys.ids_ready();
  for (int n = 0; n < S && n < my_n; ++n) issue(n);
#pragma unroll
  for (int r = 0; r < NR; ++r)
#pragma unroll
    for (int kk = 0; kk < C::KK; ++kk) asm volatile("" ::"v"(qf[r][kk]));
  for (int n = 0; n < my_n; ++n) {
    const int pos0 = first_pos + kStep * n, rem = my_n - 1 - n;
    const unsigned char* stage = stages + n % S * C::TILE_BYTES;
    // Behind the tile are those of the next S - 1, and from iteration S + 1 on the stores of S iterations
    // (memory instructions retire in order): a wait that left those out would be one for the next tile. The
    // last and the first iterations wait for more than they need, and those of more rows than the count says.
    if (rem >= S - 1 && n > S && it.rows <= 8)
      wait_vm<(S - 1) * C::INSTR + S>();
    else if (rem >= S - 1 && n > S && it.rows <= 16)
      wait_vm<(S - 1) * C::INSTR + 2 * S>();
    else if (rem >= S - 1 && n > S && (NR == 1 || it.rows <= 32))
      wait_vm<(S - 1) * C::INSTR + 3 * S>();
    else if (rem >= S - 1 && n > S)
      wait_vm<(S - 1) * C::INSTR + 5 * S>();
    else if (rem >= S - 1)
      wait_vm<(S - 1) * C::INSTR>();
    else
      wait_vm<0>();
    asm volatile("" ::: "memory");
    u32x4 ka[C::KK];
#pragma unroll
    for (int kk = 0; kk < C::KK; ++kk) ka[kk] = read_k<C>(stage, ln, 0, kk);
    wait_lds();
    __builtin_amdgcn_sched_barrier(0);
    if (rem >= S) issue(n + S);
    f32x16 s[NR][1];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      f32x16 t;
#pragma unroll
      for (int v = 0; v < 16; ++v) s[r][0][v] = t[v] = 0.0f;
#pragma unroll
      for (int kk = 0; kk < C::KK; kk += 2) {
        s[r][0] = Elem<C::BF16>::mma(ka[kk], qf[r][kk], s[r][0]);
        t = Elem<C::BF16>::mma(ka[kk + 1], qf[r][kk + 1], t);
      }
      s[r][0] += t;
      if (pos0 + C::BN > hi_min) mask_seen<C>(s[r], pos0, seen[r], hh);
      float sum = exp_sum(s[r][0], m[r], p.scale_log2);
      if (__ballot(!(sum <= kSoftmaxSumBound))) {
        const float top = fmaxf(m[r], row_max<C>(s[r], p.scale_log2));
        l[r] *= __builtin_amdgcn_exp2f(m[r] - top);
        m[r] = top;
        sum = exp_sum(s[r][0], top, p.scale_log2);
      }
      l[r] += sum;
    }
    if (n > 0) store_kept(pos0 - kStep);
    wave_fence();
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      if (32 * r + il < it.rows) {
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4*>(&out[wave][(32 * r + il) * kRow + 8 * g + 4 * hh]) =
              f32x4{s[r][0][4 * g], s[r][0][4 * g + 1], s[r][0][4 * g + 2], s[r][0][4 * g + 3]} * p.scale_log2;
      }
    }
    wave_fence();
  }
  if (my_n > 0) store_kept(first_pos + kStep * (my_n - 1));

#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const float tot = pair_sum(l[r]);
    if (hh == 0 && 32 * r + il < it.rows) {
      cm[wave * ROWS + 32 * r + il] = m[r];
      cl[wave * ROWS + 32 * r + il] = tot;
    }
  }
  wait_vm<0>();  // the kept scores of every wave
  __syncthreads();
  if (tid < it.rows) {
    float mm = kNegBig, t2 = 0.0f;
#pragma unroll
    for (int k = 0; k < C::NWK; ++k) mm = fmaxf(mm, cm[k * ROWS + tid]);
#pragma unroll
    for (int k = 0; k < C::NWK; ++k) t2 += cl[k * ROWS + tid] * __builtin_amdgcn_exp2f(cm[k * ROWS + tid] - mm);
    const float lse = lse2_of(mm, t2);
    clse[tid] = lse;
    if (it.splits > 1) p.lse[(int64_t)it.slot * ROWS + tid] = lse;
  }
  if (it.splits > 1) return;
  __syncthreads();
  finish_keys(p, it, clse, 0, it.len, tid, C::THREADS);
}

// The items of weights_rows_kernel again, those of split tiles.
constexpr int kFinishThreads = 256;
template <int NR>
__global__ __launch_bounds__(kFinishThreads) void weights_finish_kernel(WeightParams p, const int32_t* __restrict__ lengths,
                                                                       const int32_t* __restrict__ cu) {
  constexpr int ROWS = 32 * NR, kShare = kFinishThreads / ROWS;
  __shared__ float part[kFinishThreads], clse[ROWS];
  const int tid = threadIdx.x;
  Item it;
  if (!find_item<KeptTiling<NR>>(p, lengths, cu, (int)blockIdx.x, tid & 63, it) || it.splits == 1) return;
  // kShare threads to a row, then its first one.
  const int r = tid % ROWS, g = tid / ROWS;
  float m = kNegBig, l = 0.0f;
  if (r < it.rows) {
    for (int s = g; s < it.splits; s += kShare) {
      const float x = p.lse[(int64_t)(it.slot0 + s * it.slot_step) * ROWS + r], top = fmaxf(m, x);
      l = l * __builtin_amdgcn_exp2f(m - top) + __builtin_amdgcn_exp2f(x - top);
      m = top;
    }
  }
  part[tid] = l > 0.0f || l != l ? lse2_of(m, l) : kNegBig;
  __syncthreads();
  if (tid < it.rows) {
    float top = kNegBig, sum = 0.0f;
    for (int k = 0; k < kShare; ++k) top = fmaxf(top, part[k * ROWS + tid]);
    for (int k = 0; k < kShare; ++k) sum += __builtin_amdgcn_exp2f(part[k * ROWS + tid] - top);
    clse[tid] = lse2_of(top, sum);
  }
  __syncthreads();
  const int from = it.blk_begin * KeptTiling<NR>::BN, to = it.blk_end * KeptTiling<NR>::BN;
  finish_keys(p, it, clse, from, to < it.len ? to : it.len, tid, kFinishThreads);
}

// ---- more rows ----------------------------------------------------------------------------------

// Waves that share tiles of 64 keys or rows in LDS, each with NR times 32 rows or keys of its own, 256 in all.
template <bool BF16_, int DPAD_>
struct WCfg {
  static constexpr bool BF16 = BF16_;
  static constexpr int DPAD = DPAD_, NWQ = DPAD == 256 ? 8 : 4, NWK = 1, BN = 64, THREADS = 64 * NWQ;
  static constexpr int NR = DPAD == 256 ? 1 : 2, ROWS_WAVE = 32 * NR, ROWS_TILE = NWQ * ROWS_WAVE;
  static constexpr int KK = DPAD / 16, ST = BN / 32, CPR = DPAD / 8, ROW_BYTES = DPAD * 2;
  static constexpr int TILE_BYTES = BN * ROW_BYTES, INSTR = TILE_BYTES / 1024, INSTR_PER_WAVE = INSTR / NWQ;
  static constexpr int KSW = CMin<16, CPR>::value, VSW = CPR / 4, RPI = 64 / CPR;
  static constexpr int STAGES = 3;
  static_assert(ROWS_TILE == 256 && DPAD >= 64 && INSTR_PER_WAVE >= 1 && ST * NR % 2 == 0, "DMA granularity");
};
template <class C>
struct OneTile {  // of mask_seen and row_max: 32 rows
  static constexpr int ST = 1;
};

// The loop of both kernels. A step is a tile of 64 in LDS against the wave's own 32 NR: ST * NR products of
// 32 x 32, phase (t, r) its rows 32 t .. against the wave's 32 r .. . The matrix and the vector unit run side
// by side only where their instructions come by turns (16 products 222 ns, the 32 exponentials of a lane with
// their sums 221 ns; by turns 277 to 333, one after the other 443), so between a phase's products stand the
// exponentials of the phase before: use(s, t, r, e) takes element e of it; begin(j, s, t, r) and end(s, t, r)
// come before and after. issue(j, lds offset) starts tile j's DMA (start_tiles: that of the first ones). begin says whether the phase takes the
// common path; if not, rare(s, t, r) stands for all its elements.
template <class C, class Issue>
__device__ __forceinline__ void start_tiles(int tiles, Issue&& issue) {
  for (int j = 0; j < C::STAGES - 1 && j < tiles; ++j) issue(j, j * C::TILE_BYTES);
}
template <class C, class Issue, class Begin, class Use, class Rare, class End>
__device__ __forceinline__ void stream_tiles(int tiles, u32 lds, const Lanes<C>& ln, const u32x4 (&held)[C::NR][C::KK],
                                             Issue&& issue, Begin&& begin, Use&& use, Rare&& rare, End&& end) {
  using E = Elem<C::BF16>;
  // (Operands: those of all 32 rows up to D 128, where the NR phases share them; at D 256, where all would leave
  // too few registers, eight ahead.)
  constexpr int kAhead = C::STAGES - 1, PH = C::ST * C::NR, RING = C::KK < 8 ? C::KK : 8;
  static_assert(C::NR == 1 || RING == C::KK, "phases share their operands");
  if (tiles <= 0) return;
  u32 addr[C::KK];
#pragma unroll
  for (int kk = 0; kk < C::KK; ++kk) addr[kk] = lds + (u32)(ln.k_base + 32 * (kk ^ ln.ky));
  u32x4 a[RING];
  f32x16 s[2][1];
  auto read = [&](auto t, auto kk, u32 at) {
    constexpr int T = decltype(t)::value, K = decltype(kk)::value;
    a[K % RING] = *(const __attribute__((address_space(3))) u32x4*)(lds_at(addr[K]) + at + T * 32 * C::ROW_BYTES);
  };
  int stage = 0;
  for (int j = 0; j < tiles; ++j) {
    if (kAhead > 1 && j + 1 < tiles)
      wait_vm<(kAhead - 1) * C::INSTR_PER_WAVE>();
    else
      wait_vm<0>();
    __syncthreads();  // tile j has landed for all waves, tile j - 1 is read
    const u32 at = (u32)(stage * C::TILE_BYTES);
    static_for<RING>([&](auto kk) { read(std::integral_constant<int, 0>{}, kk, at); });
    if (j + kAhead < tiles) issue(j + kAhead, (stage == 0 ? C::STAGES - 1 : stage - 1) * C::TILE_BYTES);
    static_for<PH>([&](auto ph) {
      constexpr int P = decltype(ph)::value, T = P / C::NR, R = P % C::NR, Q = (P + PH - 1) % PH, QT = Q / C::NR, QR = Q % C::NR;
      f32x16(&next)[1] = s[P % 2];
      f32x16(&cur)[1] = s[(P + 1) % 2];
      auto products = [&](auto&& between) {
#pragma unroll
        for (int v = 0; v < 16; ++v) next[0][v] = 0.0f;
        static_for<C::KK>([&](auto kk) {
          constexpr int K = decltype(kk)::value;
          next[0] = E::mma(a[K % RING], held[R][K], next[0]);
          if constexpr (K + RING < C::KK)
            read(std::integral_constant<int, T>{}, std::integral_constant<int, K + RING>{}, at);
          else if constexpr (R == C::NR - 1 && T + 1 < C::ST)
            read(std::integral_constant<int, T + 1>{}, std::integral_constant<int, K + RING - C::KK>{}, at);
          if constexpr (K > 0) between(K - 1);  // (the phase before's last product is through by then)
          __builtin_amdgcn_sched_barrier(0);
        });
        between(C::KK - 1);
        __builtin_amdgcn_sched_barrier(0);
      };
      if (P > 0 || j > 0) {
        if (begin(P > 0 ? j : j - 1, cur, QT, QR)) {
          products([&](int k) {
#pragma unroll
            for (int e = 16 * k / C::KK; e < 16 * (k + 1) / C::KK; ++e) use(cur[0], QT, QR, e);
          });
        } else {
          products([](int) {});
          rare(cur[0], QT, QR);
        }
        end(cur, QT, QR);
      } else {
        products([](int) {});
      }
    });
    stage = stage + 1 == C::STAGES ? 0 : stage + 1;
  }
  f32x16(&cur)[1] = s[1];
  if (begin(tiles - 1, cur, C::ST - 1, C::NR - 1)) {
#pragma unroll
    for (int e = 0; e < 16; ++e) use(cur[0], C::ST - 1, C::NR - 1, e);
  } else {
    rare(cur[0], C::ST - 1, C::NR - 1);
  }
  end(cur, C::ST - 1, C::NR - 1);
}

template <class C>
__global__ __launch_bounds__(C::THREADS, kWaveSimd) void weights_stats_kernel(
    WeightParams p, const int32_t* __restrict__ table, const int32_t* __restrict__ lengths, const int32_t* __restrict__ cu) {
  typedef StatsTiling T;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[C::STAGES * C::TILE_BYTES];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int il = lane & 31, hh = lane >> 5;
  Item it;
  int chunk;
  if (!find_item<T>(p, lengths, cu, (int)blockIdx.x, lane, it, &chunk)) return;
  if (it.place == 0 && it.head == 0 && tid == 0)
    reinterpret_cast<WeightNote*>(p.request_notes)[it.b] = WeightNote{(int)blockIdx.x / p.heads, it.place_splits, it.tiles, chunk};
  const int first_pos = it.blk_begin * T::BN, tiles = it.blk_end - it.blk_begin;
  KeyStream<C, false> keys(p, table, it, lane, wave, first_pos, C::BN, tiles);
  const DmaLanes<C> dl(lane, wave, keys.row_bytes);
  const u32 lds = lds_address(smem);
  const Lanes<C> ln(lane);
  u32x4 qf[C::NR][C::KK];
  int in_tile[C::NR], hi_min[C::NR];
  Seen seen[C::NR];
  float m[C::NR], l[C::NR], rs[4];
#pragma unroll
  for (int r = 0; r < C::NR; ++r) {
    in_tile[r] = wave * C::ROWS_WAVE + 32 * r + il;
    const int row = it.tile * C::ROWS_TILE + in_tile[r];
    load_q<C>(p, it, row, in_tile[r] < it.rows, hh, qf[r]);
    seen[r] = row_seen(p, it, row / p.group);
    hi_min[r] = row_seen(p, it, (it.tile * C::ROWS_TILE + wave * C::ROWS_WAVE + 32 * r) / p.group).hi;
    m[r] = kNegBig;
    l[r] = 0.0f;
  }
  keys.ids_ready();
  auto issue_tile = [&](int j, int at) { keys.template issue<false>(dl, j, lds + (u32)at); };
  start_tiles<C>(tiles, issue_tile);
#pragma unroll
  for (int r = 0; r < C::NR; ++r)
#pragma unroll
    for (int kk = 0; kk < C::KK; ++kk) asm volatile("" ::"v"(qf[r][kk]));
  stream_tiles<C>(
      tiles, lds, ln, qf, issue_tile,
      [&](int j, f32x16(&s)[1], int t, int r) {
        const int pos0 = first_pos + C::BN * j + 32 * t;
        if (pos0 + 32 > hi_min[r]) mask_seen<OneTile<C>>(s, pos0, seen[r], hh);
        return true;
      },
      [&](const f32x16& s, int, int r, int e) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], p.scale_log2, -m[r]));
        rs[e % 4] = e < 4 ? x : rs[e % 4] + x;
      },
      [](const f32x16&, int, int) {},
      [&](const f32x16(&s)[1], int, int r) {
        float sum = (rs[0] + rs[1]) + (rs[2] + rs[3]);
        if (__ballot(!(sum <= kSoftmaxSumBound))) {
          const float top = fmaxf(m[r], row_max<OneTile<C>>(s, p.scale_log2));
          l[r] *= __builtin_amdgcn_exp2f(m[r] - top);
          m[r] = top;
          sum = exp_sum(s[0], top, p.scale_log2);
        }
        l[r] += sum;
      });
#pragma unroll
  for (int r = 0; r < C::NR; ++r) {
    const float tot = pair_sum(l[r]);
    if (hh == 0 && in_tile[r] < it.rows) p.lse[(int64_t)it.slot * C::ROWS_TILE + in_tile[r]] = lse2_of(m[r], tot);
  }
}

// Items of the other two kernels. weights_columns_kernel: the parts of a request's rows, the last first,
// each with the blocks of keys that some row of it sees (the more, the later the part). weights_sum_kernel:
// blocks of keys of the requests with several parts.
struct Column {
  int b, head, first, n, len, from, block, part, parts, part0;
};
// Blocks of kColumnKeys keys that the rows of a part see: up to its last row's token.
__device__ __forceinline__ int blocks_seen(const WeightParams& p, int n, int len, int part) {
  const int64_t rows = (int64_t)n * p.group, end = (int64_t)(part + 1) * p.part_rows;
  const int last = (int)((u32)((end < rows ? end : rows) - 1) / (u32)p.group), hi = len - n + last + 1;
  return hi > 0 ? (hi + kColumnKeys - 1) / kColumnKeys : 0;
}
// Those of a launch among the first `blocks`.
__device__ __forceinline__ int blocks_here(const WeightParams& p, int blocks) {
  const int to = blocks < p.block_to ? blocks : p.block_to;
  return to > p.block_from ? to - p.block_from : 0;
}
struct ColumnRequest {
  Request r;
  int parts, items;
  int places;  // for partial sums: none where one part has all rows
};
template <bool SUM>
__device__ __forceinline__ ColumnRequest column_request(const WeightParams& p, const int32_t* lengths, const int32_t* cu, int b) {
  ColumnRequest x;
  x.r = load_request<StatsTiling>(p, lengths, cu, b);
  x.parts = x.r.tiles ? (int)(((int64_t)x.r.n * p.group + p.part_rows - 1) >> p.part_shift) : 0;
  x.places = x.parts > 1 ? x.parts : 0;
  x.items = 0;
  if (SUM)
    x.items = x.parts > 1 ? blocks_here(p, (x.r.len + kColumnKeys - 1) / kColumnKeys) : 0;
  else
    for (int c = 0; c < x.parts; ++c) x.items += blocks_here(p, blocks_seen(p, x.r.n, x.r.len, c));
  return x;
}
template <bool SUM>
__device__ __forceinline__ bool find_column(const WeightParams& p, const int32_t* lengths, const int32_t* cu, int64_t w,
                                            int lane, const ColumnRequest& x0, Column& it) {
  const int64_t g = w / p.heads;
  it.head = (int)(w - g * p.heads);
  int64_t before = 0;
  int places_before = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 64) {
    const ColumnRequest x = b0 == 0 ? x0 : column_request<SUM>(p, lengths, cu, b0 + lane);
    const int items_to = wave_incl_sum(x.items, lane), places_to = wave_incl_sum(x.places, lane);
    const int64_t at = g - before - (items_to - x.items);
    const uint64_t hit = __ballot(at >= 0 && at < x.items);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      auto pick = [&](int y) { return __builtin_amdgcn_readlane(y, l); };
      it.b = b0 + l;
      it.first = pick(x.r.first);
      it.n = pick(x.r.n);
      it.len = pick(x.r.len);
      it.from = pick(x.r.from);
      it.parts = pick(x.parts);
      it.part0 = places_before + pick(places_to - x.places);
      it.block = p.block_from + pick((int)at);
      it.part = 0;
      if (SUM || it.parts == 1) return true;
      for (int c0 = 0; c0 < it.parts; c0 += 64) {  // the part: one to a lane
        const int c = it.parts - 1 - c0 - lane, n = c >= 0 ? blocks_here(p, blocks_seen(p, it.n, it.len, c)) : 0;
        const int to = wave_incl_sum(n, lane);
        const uint64_t here = __ballot(it.block - p.block_from < to);
        if (here) {
          const int k = __builtin_ctzll(here);
          it.part = it.parts - 1 - c0 - k;
          it.block -= __builtin_amdgcn_readlane(to - n, k);
          return true;
        }
        it.block -= __builtin_amdgcn_readlane(to, 63);
      }
      return false;
    }
    before += __builtin_amdgcn_readlane(items_to, 63);
    places_before += __builtin_amdgcn_readlane(places_to, 63);
  }
  return false;
}
// The first row of a request that sees the key (rows see their token's own position and all before it); past
// the last row, where none does.
__device__ __forceinline__ int first_row(const WeightParams& p, const Column& it, int key) {
  const int token = key - (it.len - it.n);
  return token > 0 ? (token < it.n ? token : it.n) * p.group : 0;
}

template <class C>
__global__ __launch_bounds__(C::THREADS, kWaveSimd) void weights_columns_kernel(
    WeightParams p, const int32_t* __restrict__ table, const int32_t* __restrict__ lengths, const int32_t* __restrict__ cu) {
  __shared__ __attribute__((aligned(1024))) unsigned char smem[C::STAGES * C::TILE_BYTES];
  __shared__ __attribute__((aligned(16))) float slse[kColumnRows + 64];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int il = lane & 31, hh = lane >> 5;
  const u32 lds = lds_address(smem);
  const Lanes<C> ln(lane);
  const ColumnRequest r0 = column_request<false>(p, lengths, cu, lane);
  const int64_t row_bytes = (int64_t)p.heads * p.dim * 2;
  Column it;
  for (int64_t w = blockIdx.x; find_column<false>(p, lengths, cu, w, lane, r0, it); w += gridDim.x) {
    const int rows = it.n * p.group, key0 = it.block * kColumnKeys + wave * C::ROWS_WAVE;  // keys of this wave
    const int end = rows - it.part * p.part_rows < p.part_rows ? rows : (it.part + 1) * p.part_rows;
    // (Tiles of 64 rows from the part's first row.)
    const int part0 = it.part * p.part_rows, seen0 = first_row(p, it, it.block * kColumnKeys);
    if (seen0 >= end) continue;
    const int begin = seen0 > part0 ? part0 + (seen0 - part0) / 64 * 64 : part0, tiles = (end - begin + 63) / 64;

    __syncthreads();  // the item before is done with slse and the stages
    // 64 rows of Q into LDS, a K tile's layout, tile after tile: a lane's rows are 64 apart, so their places
    // move on by whole tokens and a few heads.
    constexpr int U = C::INSTR_PER_WAVE;
    const int hop = C::BN / p.group, skip = C::BN - hop * p.group;  // tokens and heads of 64 rows
    const int64_t hop_bytes = hop * p.q_token + skip * p.q_head, wrap_bytes = p.q_token - p.group * p.q_head;
    const char* src[U];
    int src_head[U], next_row = begin + C::RPI * wave + lane / C::CPR;  // (of instruction 0)
    constexpr int kApart = C::RPI * C::NWQ;                             // rows between instructions
    u32 live_dims = 0;  // instruction q's chunk lies below D
#pragma unroll
    for (int q = 0; q < U; ++q) {
      const int i = q * C::NWQ + wave, r = C::RPI * i + lane / C::CPR, row = begin + r, c = lane % C::CPR ^ (r % C::KSW);
      const int token = (int)((u32)row / (u32)p.group);
      src_head[q] = row - token * p.group;
      live_dims |= c * 8 < p.dim ? 1u << q : 0u;
      src[q] = static_cast<const char*>(p.q) + (int64_t)(it.first + token) * p.q_token +
               (int64_t)(it.head * p.group + src_head[q]) * p.q_head + c * 16;
    }
    // Places behind the part's rows take its last row again, which weighs nothing there (its L is infinite): zeros
    // would give NaN beside a key that holds an infinity. They are in a request's last part alone, and its
    // last row sees every key, so what is NaN with it is NaN in any case.
    static_assert(kApart % C::KSW == 0 && kColumnRows / 4 % C::BN == 0, "a lane's chunk is the same in all its rows");
    const char* const last_row = static_cast<const char*>(p.q) + (int64_t)(it.first + it.n - 1) * p.q_token +
                                 (int64_t)(it.head * p.group + p.group - 1) * p.q_head +
                                 (lane % C::CPR ^ (C::RPI * wave + lane / C::CPR) % C::KSW) * 16;
    auto issue_tile = [&](int, int at) {
      const char* zero = reinterpret_cast<const char*>(kZeroChunk);
#pragma unroll
      for (int q = 0; q < U; ++q) {
        const char* const row = next_row < end - q * kApart ? src[q] : last_row;
        dma_flat(p.dim == C::DPAD || (live_dims >> q & 1u) ? row : zero, lds + (u32)at + 1024u * (u32)(q * C::NWQ + wave));
        src_head[q] += skip;
        const bool wrap = src_head[q] >= p.group;
        src_head[q] -= wrap ? p.group : 0;
        src[q] += hop_bytes + (wrap ? wrap_bytes : 0);
      }
      next_row += C::BN;
    };
    start_tiles<C>(tiles, issue_tile);

    // K of the lane's keys, from their pages.
    u32x4 kf[C::NR][C::KK];
    int mine[C::NR], all[C::NR];  // the first row that sees the lane's key, all of the wave's 32
#pragma unroll
    for (int r = 0; r < C::NR; ++r) {
      const int key = key0 + 32 * r + il;
      const u32 pg = key < it.len ? div_page((u32)key, p.page_magic, p.page_shift) : 0u;
      const int64_t krow = (int64_t)table[(int64_t)it.b * p.width + pg] * p.page_size + ((u32)key - pg * (u32)p.page_size);
      const bool live = key < it.len && krow >= 0 && krow < p.pool_rows;
      const char* const kp = static_cast<const char*>(p.k) + (int64_t)it.head * p.dim * 2 + (live ? krow * row_bytes : 0);
#pragma unroll
      for (int kk = 0; kk < C::KK; ++kk) {
        const int d = 16 * kk + 8 * hh;
        u32x4 x = {0u, 0u, 0u, 0u};
        if (live && d < p.dim) x = *reinterpret_cast<const u32x4*>(kp + 2 * d);
        kf[r][kk] = x;
      }
      mine[r] = first_row(p, it, key);
      all[r] = first_row(p, it, key0 + 32 * r + 31);
    }
    // L of the part's rows, from their splits.
    const WeightNote note = reinterpret_cast<const WeightNote*>(p.request_notes)[it.b];
    // (Threads that the rows leave over share a row's splits.)
    const int padded = C::BN * tiles, share = padded < C::THREADS ? C::THREADS / padded : 1;
    for (int base = 0; base < padded; base += C::THREADS) {
      const int in_part = share > 1 ? tid % padded : base + tid, g = share > 1 ? tid / padded : 0, r = begin + in_part;
      float m = kNegBig, l = 0.0f;
      if (r < end && g < share) {
        typedef StatsTiling T;
        const int tile = r / T::ROWS, last = (tile + 1) * T::ROWS < rows ? (tile + 1) * T::ROWS : rows;
        int hi = it.len - it.n + (int)((u32)(last - 1) / (u32)p.group) + 1;
        hi = hi < 0 ? 0 : hi;
        const int most = splits_of(p, (hi + T::KEYS - 1) / T::KEYS, note.chunk);
        const int64_t slot = (int64_t)(note.base + (note.tiles - 1 - tile) * note.splits) * p.heads + it.head;
        int splits = most < note.splits ? most : note.splits;
        splits = slot >= 0 && slot + (int64_t)(splits - 1) * p.heads < p.work ? splits : 0;
        const float* const lse = p.lse + slot * T::ROWS + (r - tile * T::ROWS);
        const int64_t step = (int64_t)p.heads * T::ROWS;
        for (int s0 = g; s0 < splits; s0 += 8 * share) {
          float x[8], top = m;
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] = s0 + k * share < splits ? lse[(s0 + k * share) * step] : kNegBig;
#pragma unroll
          for (int k = 0; k < 8; ++k) top = fmaxf(top, x[k]);
          l *= __builtin_amdgcn_exp2f(m - top);
#pragma unroll
          for (int k = 0; k < 8; ++k) l += s0 + k * share < splits ? __builtin_amdgcn_exp2f(x[k] - top) : 0.0f;
          m = top;
        }
      }
      if (share > 1) {  // uniform; one pass
        slse[tid] = m;
        slse[C::THREADS + tid] = l;
        __syncthreads();
        if (g == 0) {
          float top = m;
          for (int k = 1; k < share; ++k) top = fmaxf(top, slse[k * padded + in_part]);
          l *= __builtin_amdgcn_exp2f(m - top);
          for (int k = 1; k < share; ++k)
            l += slse[C::THREADS + k * padded + in_part] * __builtin_amdgcn_exp2f(slse[k * padded + in_part] - top);
          m = top;
        }
        __syncthreads();
      }
      // (Rows that are none, or see nothing, weigh nothing.)
      if (g == 0 && in_part < padded) slse[in_part] = r < end && (m > 0.5f * kNegBig || l != l) ? lse2_of(m, l) : INFINITY;
    }
#pragma unroll
    for (int r = 0; r < C::NR; ++r)
#pragma unroll
      for (int kk = 0; kk < C::KK; ++kk) asm volatile("" ::"v"(kf[r][kk]));
    __syncthreads();

    float acc[C::NR][4];
#pragma unroll
    for (int r = 0; r < C::NR; ++r)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[r][k] = 0.0f;
    f32x4 lse[4];  // of the lane's rows of a phase
    int row0 = 0;  // of the phase, in the part
    stream_tiles<C>(
        tiles, lds, ln, kf, issue_tile,
        [&](int j, f32x16(&)[1], int t, int r) {
          row0 = C::BN * j + 32 * t;
          if (r == 0) {
#pragma unroll
            for (int g = 0; g < 4; ++g) lse[g] = *reinterpret_cast<const f32x4*>(slse + row0 + 8 * g + 4 * hh);
          }
          return begin + row0 >= all[r];
        },
        [&](const f32x16& s, int, int r, int e) {
          acc[r][e % 4] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], p.scale_log2, -lse[e / 4][e % 4]));
        },
        [&](const f32x16& s, int, int r) {  // some of the wave's keys lie behind rows of the phase
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], p.scale_log2, -lse[e / 4][e % 4]));
            acc[r][e % 4] += begin + row0 + 8 * (e / 4) + 4 * hh + e % 4 >= mine[r] ? x : 0.0f;
          }
        },
        [](const f32x16(&)[1], int, int) {});
#pragma unroll
    for (int r = 0; r < C::NR; ++r) {
      const int key = key0 + 32 * r + il;
      const float sum = pair_sum((acc[r][0] + acc[r][1]) + (acc[r][2] + acc[r][3]));
      if (hh == 0 && key < it.len) {
        if (it.parts == 1)
          add_score(p, p.scores + ((int64_t)it.b * p.heads + it.head) * p.stride, key, it.from, sum);
        else if (it.part0 + it.part < p.parts_most)
          p.sums[((int64_t)(it.part0 + it.part) * p.heads + it.head) * p.keys_pad + (key - p.block_from * kColumnKeys)] = sum;
      }
    }
  }
}

static __global__ __launch_bounds__(kFinishThreads) void weights_sum_kernel(WeightParams p, const int32_t* __restrict__ lengths,
                                                                           const int32_t* __restrict__ cu) {
  const int tid = threadIdx.x, lane = tid & 63;
  const ColumnRequest r0 = column_request<true>(p, lengths, cu, lane);
  Column it;
  for (int64_t w = blockIdx.x; find_column<true>(p, lengths, cu, w, lane, r0, it); w += gridDim.x) {
    const int end = it.len < (it.block + 1) * kColumnKeys ? it.len : (it.block + 1) * kColumnKeys;
    float* const row = p.scores + ((int64_t)it.b * p.heads + it.head) * p.stride;
    for (int key = it.block * kColumnKeys + tid; key < end; key += kFinishThreads) {
      // Parts whose rows all come before the key's block left nothing.
      float sum = 0.0f;
      const int last = it.part0 + it.parts < p.parts_most ? it.part0 + it.parts : p.parts_most;
      const float* const at = p.sums + (int64_t)it.head * p.keys_pad + (key - p.block_from * kColumnKeys);
      const int64_t step = (int64_t)p.heads * p.keys_pad;
      int c = it.part0 + (first_row(p, it, key / kColumnKeys * kColumnKeys) >> p.part_shift);
      for (; c + 4 <= last; c += 4) {
        float x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = at[(c + k) * step];
#pragma unroll
        for (int k = 0; k < 4; ++k) sum += x[k];
      }
      for (; c < last; ++c) sum += at[c * step];
      add_score(p, row, key, it.from, sum);
    }
  }
}

template <bool BF16, int DPAD>
hipError_t launch_weights(const WeightParams& p, bool many, int grid, hipStream_t stream) {
  if (!many) {
    using C = Cfg<BF16, DPAD, kLayoutKey, DPAD == 128 ? 1 : 0>;
    if (p.kept_rows <= 32)
      weights_rows_kernel<C, 1><<<dim3(grid), dim3(C::THREADS), 0, stream>>>(p, p.table, p.lengths, p.cu);
    else
      weights_rows_kernel<C, 2><<<dim3(grid), dim3(C::THREADS), 0, stream>>>(p, p.table, p.lengths, p.cu);
  } else {
    using C = WCfg<BF16, DPAD>;
    weights_stats_kernel<C><<<dim3(grid), dim3(C::THREADS), 0, stream>>>(p, p.table, p.lengths, p.cu);
  }
  return hipGetLastError();
}
template <bool BF16, int DPAD>
hipError_t launch_weights_columns(const WeightParams& p, int grid, hipStream_t stream) {
  using C = WCfg<BF16, DPAD>;
  weights_columns_kernel<C><<<dim3(grid), dim3(C::THREADS), 0, stream>>>(p, p.table, p.lengths, p.cu);
  return hipGetLastError();
}

}  // namespace fgw_kv
