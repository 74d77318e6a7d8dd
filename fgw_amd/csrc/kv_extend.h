// Attention of packed new tokens over the paged cache, grouped K/V heads (fgw_kv_extend).
//
// Request b has n_b new tokens, the last of its len_b cached ones; query head h reads K/V head
// h / G, G = heads / kv_heads. The G query heads of a token that share a K/V head are rows of one
// tile: row R of (request, K/V head) is token R / G, head R % G of the group, so a tile of 32 rows
// reads each key once for all of them. Row R sees the keys [lo, hi) of its token:
//   hi = len - n + token + 1 (causal; else len),  lo = hi - window (no window: 0).
// Softmax and products are those of fmha_kernel.h (fp32 sums and statistics). For the PV product P is
// two numbers of the input type in the kernel of few rows, which memory bounds, and one (rounded) in
// the kernels of long tiles: there the second product would be half as many matrix operations again
// where those are the bound. Error against 64 bits relative to the output (q of standard deviation 2,
// the rest 1; the output's own rounding alone 0.0017 in BF16, 0.00021 in FP16): one number
// 0.0022-0.0023 and 0.00027, two as the rounding alone; 4096 tokens, Hq 32, Hkv 8, D 256 take 424 us
// with one, 796 with two.
//
// Work. Lengths and counts are on the device, so each program finds its item itself (find_item): it
// reads the lengths of 64 requests at a time, one to a lane, and sums tiles and splits over the
// wave. An item is a tile, or where tiles are fewer than the `target` programs that fill the card,
// one of its splits: a tile of u units of keys has ceil(u / chunk) of them, with the smallest chunk
// that leaves no more than `target` items (best_chunk). So all items run at once, the long requests
// of a ragged batch in pieces. A CU that reads alone takes 32 GB/s at D 64, 42 at D 128 and 48 at D
// 256, where its share of the memory is 20: pieces of unequal length cost little until one has twice
// its share (B 32, Hq 32, Hkv 8, D 128, lengths 1024-4096, one tile to a CU, us: whole tiles 68.7,
// split evenly by W / target 74.6; see also extend_rows_kernel). Grid and workspace follow on the host
// from sizes alone, programs without an item end after the sums. Split tiles go through partials
// (O / l, LSE) and a join.
// The K/V head is fastest in an item's number: workgroup w runs on XCD w % 8, so with 8 heads an XCD
// holds one of them.
#pragma once
#include "fmha_prefill.h"

namespace fgw_kv {

using namespace fgw_mha;

// heads: K/V heads; work: places for partials; sq, q_tiles, mode, splits: unused.
struct ExtendParams : FwdParams {
  const int32_t* cu;
  int64_t q_token, q_head;  // bytes
  int32_t tokens, q_heads, group, max_new, window;
  int32_t rows_from, rows_to;  // requests with n * group in (rows_from, rows_to] are this launch's
  int32_t target, min_chunk;   // items that fill the card (0: nothing is split), units of a split at least
  int32_t whole, many;         // units of a tile that is never split, that has splits of 2 min_chunk
  int32_t* counters;           // rows kernel: arrivals at the split tiles, by their first item, or nullptr
  int32_t* notes;              // for the join: [work] JoinNote
};

// Requests in groups that share a prefix (fgw_kv_shared; kv_shared.hip has the two passes). The first
// pass attends over the groups' prefixes, each a request of the kernels below whose rows are those of all
// its group's tokens, and leaves partials; the second over the rest of each request's keys, and joins.
struct SharedParams : ExtendParams {
  const int32_t* groups;    // [n_groups + 1]
  const int32_t* prefixes;  // [n_groups]
  int32_t n_groups;
  int32_t prefix_slots, prefix_rows;  // places of the first pass's partials, rows of a place
  const float* prefix_parts;
  const float* prefix_lse;
  int32_t* group_notes;     // [n_groups] GroupNote
  int32_t share_from;       // units of 64 KB that sharing has to gain (Requests::pays); 0: it always pays
};
struct PrefixParams : SharedParams {};
struct SuffixParams : SharedParams {};
template <class P>
constexpr bool kIsPrefix = std::is_same<P, PrefixParams>::value;
template <class P>
constexpr bool kIsSuffix = std::is_same<P, SuffixParams>::value;
template <class P>
constexpr bool kPicksFrom = kIsSuffix<P>;  // items with Request::from

// Where a group's partials are: those of its first item (a place for each K/V head), the splits of its
// tiles, how many tiles, and the group's first token. Written by the first pass.
struct GroupNote {
  int32_t base, splits, tiles, first;
};
constexpr int kShareRows = 128;  // of a request, on average over its group, up to which sharing may pay
// What the first pass costs for a row that shares, as bytes of reading for each of its dims (kv_shared.hip).
constexpr int kShareDimBytes = 340;

// Tiles of ROWS rows, keys in blocks of BN, splits in units of UNIT blocks.
template <int ROWS_, int BN_, int UNIT_>
struct Tiling {
  static constexpr int ROWS = ROWS_, BN = BN_, UNIT = UNIT_, KEYS = BN_ * UNIT_;
};
typedef Tiling<32, 32, 4> ShortTiling;   // extend_rows_kernel: a round of its four waves
typedef Tiling<256, 64, 1> LongTiling;   // extend_long_kernel
typedef Tiling<128, 64, 1> WideTiling;   // extend_wide_kernel

struct Request {
  int first, n, len, tiles, units;
  int row;          // prefix pass: of the block table
  int from, group;  // suffix pass: keys [0, from) are in the prefix of `group` (-1: none shared)
                    // (attention weight, kv_weights.h: keys [0, from) were there before the new tokens)
};

template <class P>
__device__ __forceinline__ int requests_of(const P& p) {
  if constexpr (kIsPrefix<P>) return p.n_groups;
  else return p.batch;
}

template <class T>
__device__ __forceinline__ Request load_request(const ExtendParams& p, const int32_t* lengths,
                                                const int32_t* cu, int b) {
  Request r{0, 0, 0, 0, 0, 0, 0, -1};
  if (b >= p.batch) return r;
  const int first = cu[b], next = cu[b + 1];
  int len = lengths[b];
  const int capacity = p.width * p.page_size;
  r.len = len < 0 ? 0 : (len > capacity ? capacity : len);
  r.first = first;
  if (first < 0 || next > p.tokens || next <= first) return r;
  r.n = next - first;
  const int count = r.n < p.max_new ? r.n : p.max_new;
  const int64_t rows = (int64_t)count * p.group;
  if (rows <= p.rows_from || rows > p.rows_to) return r;
  r.tiles = (int)((rows + T::ROWS - 1) / T::ROWS);
  int lo = p.window > 0 ? r.len - r.n - p.window + 1 : 0;
  lo = lo < 0 ? 0 : lo;
  int end = p.causal ? r.len - r.n + count : r.len;
  end = end < 0 ? 0 : end;
  r.units = (end + T::KEYS - 1) / T::KEYS - lo / T::KEYS;
  return r;
}

// Inclusive sums over the wave's lanes: by DPP within rows of 16 (shifts by 1, 2, 4, 8), then each
// row's last lane onto the rows behind it.
__device__ __forceinline__ int wave_incl_sum(int x, int lane) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  const int a = __builtin_amdgcn_readlane(x, 15), b = __builtin_amdgcn_readlane(x, 31);
  const int c = __builtin_amdgcn_readlane(x, 47);
  return x + (lane >= 16 ? a : 0) + (lane >= 32 ? b : 0) + (lane >= 48 ? c : 0);
}
__device__ __forceinline__ int wave_sum(int x, int lane) {
  return __builtin_amdgcn_readlane(wave_incl_sum(x, lane), 63);
}

// Requests [f0, f1) of group g, its tokens [first, next) and the keys that its requests share: as many as the
// first of them, whose table row holds them, has before its new tokens (none for a request alone: it reads
// its keys itself). Two rounds of reads; every place is read within the arrays.
struct Group {
  int f0, f1, keys, first, next;
};
__device__ __forceinline__ Group load_group(const SharedParams& p, const int32_t* lengths, const int32_t* cu, int g) {
  Group x{0, 0, 0, 0, 0};
  const int at = g < p.n_groups ? g : p.n_groups - 1;
  const int f0 = p.groups[at], f1 = p.groups[at + 1], wanted = p.prefixes[at];
  const bool good = g < p.n_groups && f0 >= 0 && f1 <= p.batch && f1 > f0 + 1;
  const int a = good ? f0 : 0, b = good ? f1 : 0, capacity = p.width * p.page_size;
  x.first = cu[a];
  x.next = cu[b];
  const int n = cu[a + 1] - x.first;
  int len = lengths[a];
  len = len < 0 ? 0 : (len > capacity ? capacity : len);
  const int before = n >= 0 && n < len ? len - n : 0;
  x.f0 = a;
  x.f1 = b;
  x.keys = good ? (wanted < before ? wanted : before) : 0;
  // (Offsets that run out of q leave the group no items in the first pass: its requests read their keys themselves.)
  if (x.keys < 0 || x.first < 0 || x.next > p.tokens || x.next <= x.first) x.keys = 0;
  // (Requests of whole long tiles are bound by their products, which sharing does not save: kv_shared.hip.)
  if (p.share_from > 0 && (int64_t)(x.next - x.first) * p.group > (int64_t)kShareRows * (x.f1 - x.f0)) x.keys = 0;
  return x;
}
// What the requests of a group would read of the prefix each on its own, less what the first pass takes for their
// rows, in units of 64 KB: once for every 32 rows, in tiles of 128 or 256 dims (a tile of 64 takes the kernel
// about as long as one of 128). (Rounded to integers before they are compared: the same in every kernel.)
__host__ __device__ __forceinline__ int shared_dims(int dim) { return dim <= 128 ? 128 : 256; }
__device__ __forceinline__ int group_gain(const SharedParams& p, const Group& x) {
  if (x.keys <= 0) return 0;
  const int64_t cost = (int64_t)(x.next - x.first) * p.q_heads * p.dim * kShareDimBytes >> 16;
  const float members = (float)(x.f1 - x.f0), rows = (float)(x.next - x.first) * (float)p.group / members;
  const float bytes = members * ceilf(rows * 0.03125f) * (float)x.keys * (float)p.heads * (float)shared_dims(p.dim) * 4.0f;
  return (int)fminf(bytes * (1.0f / 65536.0f), 16777216.0f) - (int)(cost < 16777216 ? cost : 16777216);
}

template <class T>
__device__ __forceinline__ Request group_request(const PrefixParams& p, const Group& x) {
  Request r{0, 0, 0, 0, 0, 0, 0, -1};
  if (x.keys == 0) return r;
  r.row = x.f0;
  r.len = x.keys;
  r.first = x.first;
  r.n = x.next - x.first;
  r.tiles = (int)(((int64_t)r.n * p.group + T::ROWS - 1) / T::ROWS);
  r.units = (r.len + T::KEYS - 1) / T::KEYS;
  return r;
}

// The group of each lane's request: up to 64 groups are held one to a lane (`mine`, loaded once) and passed
// around, more are searched for in memory (their first requests never fall).
template <class T>
__device__ __forceinline__ Request load_request(const SuffixParams& p, const int32_t* lengths, const int32_t* cu, int b,
                                                const Group& mine, bool share) {
  Request r = load_request<T>(static_cast<const ExtendParams&>(p), lengths, cu, b);
  int keys = 0, group = -1;
  if (!share) return r;
  if (p.n_groups <= 64) {
    for (int g = 0; g < p.n_groups; ++g) {
      const int f0 = __builtin_amdgcn_readlane(mine.f0, g), f1 = __builtin_amdgcn_readlane(mine.f1, g);
      const int shared = __builtin_amdgcn_readlane(mine.keys, g);
      if (b >= f0 && b < f1) {
        keys = shared;
        group = g;
      }
    }
  } else {
    int lo = 0, hi = p.n_groups;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.groups[mid] <= b) lo = mid; else hi = mid;
    }
    const Group x = load_group(p, lengths, cu, lo);
    group = lo;
    keys = b >= x.f0 && b < x.f1 ? x.keys : 0;
  }
  if (keys > 0 && r.n > 0 && r.len - r.n >= keys) {
    r.from = keys;
    r.group = group;
    r.units -= r.units > 0 ? r.from / T::KEYS : 0;
  }
  return r;
}

// The requests of a launch, 64 at a time, one to a lane: the first kHeld times 64 are read once and held.
template <class T, class P>
struct Requests {
  static constexpr int kHeld = kIsSuffix<P> ? 4 : 1;
  const P& p;
  const int32_t* const lengths;
  const int32_t* const cu;
  const int lane;
  Group mine{0, 0, 0, 0, 0};  // of the first 64, one to a lane
  bool share = true;
  Request held[kHeld];
  __device__ __forceinline__ Request load(int b) const {
    if constexpr (kIsSuffix<P>) return load_request<T>(p, lengths, cu, b, mine, share);
    else if constexpr (kIsPrefix<P>) return share ? group_request<T>(p, b < 64 ? mine : load_group(p, lengths, cu, b)) : Request{0, 0, 0, 0, 0, 0, 0, -1};
    else return load_request<T>(p, lengths, cu, b);
  }
  // Whether the groups' prefixes are worth the two passes and the partials between them; the same in every
  // program of both.
  __device__ __forceinline__ bool pays() const {
    if (p.share_from <= 0) return true;
    int total = wave_sum(group_gain(p, mine), lane);
    for (int g = 64; g < p.n_groups && total < p.share_from; g += 64)
      total += wave_sum(group_gain(p, load_group(p, lengths, cu, g + lane)), lane);
    return total >= p.share_from;
  }
  __device__ __forceinline__ Requests(const P& p_, const int32_t* lengths_, const int32_t* cu_, int lane_)
      : p(p_), lengths(lengths_), cu(cu_), lane(lane_) {
    if constexpr (kIsSuffix<P> || kIsPrefix<P>) {
      if (p.n_groups > 0) {
        mine = load_group(p, lengths, cu, lane);
        share = pays();
      }
    }
#pragma unroll
    for (int k = 0; k < kHeld; ++k)
      if (k == 0 || 64 * k < requests_of(p)) held[k] = load(64 * k + lane);
  }
  // f(first request, the lane's) for every 64, until one is true.
  template <class F>
  __device__ __forceinline__ bool each(F&& f) const {
#pragma unroll
    for (int k = 0; k < kHeld; ++k)
      if (64 * k < requests_of(p) && f(64 * k, held[k])) return true;
    for (int b0 = 64 * kHeld; b0 < requests_of(p); b0 += 64)
      if (f(b0, load(b0 + lane))) return true;
    return false;
  }
};

__device__ __forceinline__ int splits_of(const ExtendParams& p, int units, int chunk) {
  return units > chunk && units > p.whole ? (units + chunk - 1) / chunk : 1;
}

// Units of a split: the smallest chunk, up to the steps of the search, of at least min_chunk units
// with which all tiles of a head have at most target / heads splits together; kWhole where whole
// tiles are as many, however unequal: the partials of long tiles, 132 KB each at D 128, cost what the
// balance gains (tiles above the average share cut in two, us, whole / cut: B 2, Hq 8, Hkv 8, 4096
// tokens 111 / 111; B 4, 512 tokens, lengths 1024-4096, Hq 32, Hkv 8 106 / 136). One chunk serves
// all tiles, so items jump by the number of long tiles: 17 tiles with places for 32 stay whole, 16 are
// cut in two (a prompt of 1088 tokens, Hq 32, Hkv 8: the longest item 17 blocks; of 1024: 8). The sums
// saturate (kMany) so that they stay in 32 bits; the same in every program.
constexpr int kWhole = 0x40000000, kMany = 1 << 24;
template <class T, class P>
__device__ __forceinline__ int best_chunk(const P& p, const Requests<T, P>& all) {
  const int limit = (int)((u32)p.target / (u32)p.heads);
  if (limit <= 1) return kWhole;
  auto sum = [&](auto&& count) {
    int total = 0;
    all.each([&](int, const Request& r) {
      const int64_t x = r.tiles ? count(r) : 0;
      total += wave_sum((int)(x < kMany ? x : kMany), all.lane);
      total = total < kMany ? total : kMany;
      return false;
    });
    return total;
  };
  const int tiles = sum([](const Request& r) { return (int64_t)r.tiles; });
  if (tiles >= limit) return kWhole;
  const int units = sum([](const Request& r) { return (int64_t)r.tiles * r.units; });
  int chunk = (int)((u32)(units + limit - 1) / (u32)limit);
  const int least = units > p.many * tiles ? 2 * p.min_chunk : p.min_chunk;
  chunk = chunk < least ? least : chunk;
  for (;;) {
    const int items = sum([&](const Request& r) { return (int64_t)r.tiles * splits_of(p, r.units, chunk); });
    if (items <= limit || chunk >= kMany) return chunk;
    chunk += (chunk >> 3) + 1;  // (with whole tiles the items are fewer than the limit)
  }
}

// One item: the blocks [blk_begin, blk_end) of tile `tile` of request `b`, and of those the keys
// [lo, hi) that some row of the tile sees.
struct Item {
  int b, first, n, len, tile, head, split, splits;
  int rows;  // of the tile
  int lo, hi;
  int blk_begin, blk_end;
  int slot, slot0, slot_step;  // partials: of this split, of the first one; between splits
  int from, group;             // suffix pass: as Request's
  int place, place_splits, tiles;  // among the request's items of a head; splits of its tiles at most, tiles
};

// Item w of the launch; false where there is none. Uniform over the wave; every wave of a workgroup
// computes the same.
template <class T, class P>
__device__ __forceinline__ bool find_item(const P& p, const int32_t* lengths,
                                          const int32_t* cu, int w, int lane, Item& it,
                                          int* used_chunk = nullptr) {
  const Requests<T, P> all(p, lengths, cu, lane);
  const int chunk = p.target > 0 ? best_chunk<T>(p, all) : kWhole;
  if (used_chunk) *used_chunk = chunk;
  const int g = (int)((u32)w / (u32)p.heads);
  it.head = w - g * p.heads;
  int items_before = 0;
  bool found = false;
  all.each([&](int b0, const Request& r) {
    const int splits = splits_of(p, r.units, chunk);
    const int items = r.tiles * splits;
    const int items_to = wave_incl_sum(items, lane);
    const int at = g - items_before - (items_to - items);
    const uint64_t hit = __ballot(at >= 0 && at < items);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      auto pick = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
      const int s = pick(splits), place = pick(at), tiles = pick(r.tiles);
      it.b = kIsPrefix<P> ? pick(r.row) : b0 + l;
      it.from = kPicksFrom<P> ? pick(r.from) : 0;
      it.group = kIsSuffix<P> ? pick(r.group) : kIsPrefix<P> ? b0 + l : -1;
      it.place = place;
      it.place_splits = s;
      it.tiles = tiles;
      it.first = pick(r.first);
      it.n = pick(r.n);
      it.len = pick(r.len);
      // The last tiles first: causal, they are the longest.
      const int place_tile = (int)((u32)place / (u32)s);
      it.tile = tiles - 1 - place_tile;
      it.split = place - place_tile * s;
      it.slot = w;
      it.slot0 = w - it.split * p.heads;
      it.slot_step = p.heads;

      const int row0 = it.tile * T::ROWS, all = (it.n < p.max_new ? it.n : p.max_new) * p.group;
      it.rows = all - row0 < T::ROWS ? all - row0 : T::ROWS;
      const int t0 = row0 / p.group, t1 = (row0 + it.rows - 1) / p.group;
      int hi = p.causal ? it.len - it.n + t1 + 1 : it.len;
      hi = hi < 0 ? 0 : hi;
      int lo = kIsSuffix<P> ? it.from : p.window > 0 ? it.len - it.n + t0 - p.window + 1 : 0;
      lo = lo < 0 ? 0 : (lo > hi ? hi : lo);
      it.lo = lo;
      it.hi = hi;
      // The tile's own units, fewer than its request's where it ends earlier or begins later.
      const int from = lo / T::KEYS, units = (hi + T::KEYS - 1) / T::KEYS - from;
      const int most = splits_of(p, units, chunk);
      it.splits = most < s ? most : s;
      const int end = (hi + T::BN - 1) / T::BN;
      it.blk_begin = (from + split_bound(units, it.split, it.splits)) * T::UNIT;
      it.blk_end = (from + split_bound(units, it.split + 1, it.splits)) * T::UNIT;
      it.blk_end = it.blk_end < end ? it.blk_end : end;
      // (Offsets that fall and rise again make more items than there are places for partials.)
      found = it.split < it.splits && ((it.splits == 1 && !kIsPrefix<P>) || it.slot0 + (it.splits - 1) * it.slot_step < p.work);
      return true;
    }
    items_before += __builtin_amdgcn_readlane(items_to, 63);
    return false;
  });
  return found;
}

// The keys that row R of an item's tile sees.
struct Seen {
  int lo, hi;
};
template <class P>
__device__ __forceinline__ Seen row_seen(const P& p, const Item& it, int token) {
  int hi = p.causal ? it.len - it.n + token + 1 : it.len;
  hi = hi < 0 ? 0 : hi;
  if constexpr (kIsSuffix<P>) return Seen{it.from, hi};
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

// Element offset of row `row` of a request's rows of a K/V head in the output.
__device__ __forceinline__ int64_t out_row(const ExtendParams& p, const Item& it, int row) {
  const int tk = row / p.group;
  return ((int64_t)(it.first + tk) * p.q_heads + it.head * p.group + (row - tk * p.group)) * p.dim;
}

// Partials that this launch joins itself go through buffer loads and stores at device scope (sc1,
// 16 bytes to a lane): they pass by the L2s of the XCDs, which are not coherent with each other. Such a
// launch's partials are below 2^31 bytes (kMostCus in kv_extend_plan.h: 9 MB); those of a first pass over
// shared prefixes, which may be more, are joined by the next launch.
constexpr int kDeviceScope = 17;  // sc0 | sc1
__device__ __forceinline__ f32x4 device_load4(const float* base, u32 bytes) {
  const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(base), (short)0, 0x7fffffff, 0x00027000);
  return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)bytes, 0, kDeviceScope));
}
__device__ __forceinline__ float device_load1(const float* base, u32 bytes) {
  const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(base), (short)0, 0x7fffffff, 0x00027000);
  return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rsrc, (int)bytes, 0, kDeviceScope));
}
__device__ __forceinline__ void device_store4(float* base, u32 bytes, f32x4 x) {
  const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(base, (short)0, 0x7fffffff, 0x00027000);
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), rsrc, (int)bytes, 0, kDeviceScope);
}
__device__ __forceinline__ void device_store1(float* base, u32 bytes, float x) {
  const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(base, (short)0, 0x7fffffff, 0x00027000);
  __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(x), rsrc, (int)bytes, 0, kDeviceScope);
}

// LSE of a split's row; one that saw no key has kNegBig, one that met a NaN keeps it (lse_of calls that
// empty), so that the join neither drops the split nor returns zeros for the row.
__device__ __forceinline__ float part_lse(float m_log2, float total) {
  return total != total ? total : lse_of(m_log2, total);
}

// What a second launch has to know to join split tiles: every item's, in its own place (splits 0:
// no split tile's).
struct JoinNote {
  int32_t first, tile, head, rows, splits, split, group, pad;
};
template <class P>
__device__ __forceinline__ void write_note(const P& p, const Item& it, bool found) {
  const int w = (int)blockIdx.x;
  if constexpr (kIsPrefix<P>) {
    if (found && it.place == 0 && it.head == 0 && threadIdx.x == 0)
      reinterpret_cast<GroupNote*>(p.group_notes)[it.group] = GroupNote{w / p.heads, it.splits, it.tiles, it.first};
    return;
  }
  if (p.notes == nullptr || w >= p.work || threadIdx.x != 0) return;
  JoinNote note{0, 0, 0, 0, 0, 0, 0, 0};
  if (found && it.splits > 1)
    note = JoinNote{it.first, it.tile, it.head, it.rows, it.splits, it.split, it.group, 0};
  reinterpret_cast<JoinNote*>(p.notes)[w] = note;
}

// The partials that the first pass left for a row of a request: split s at place `slot` + s * step, row
// `row` of it.
struct PrefixRow {
  int slot, step, splits, row;
};
__device__ __forceinline__ PrefixRow prefix_row(const SharedParams& p, const GroupNote& note, int first, int head, int row) {
  const int r = (first - note.first) * p.group + row, tile = (int)((u32)r / (u32)p.prefix_rows);
  PrefixRow x;
  x.slot = (note.base + (note.tiles - 1 - tile) * note.splits) * p.heads + head;
  x.step = p.heads;
  x.row = r - tile * p.prefix_rows;
  // (Places that a group of broken offsets would not have are not read.)
  const int64_t last = (int64_t)x.slot + (int64_t)(note.splits - 1) * x.step;
  x.splits = r >= 0 && note.splits > 0 && x.slot >= 0 && last < p.prefix_slots ? note.splits : 0;
  return x;
}
__device__ __forceinline__ GroupNote group_note(const SharedParams& p, int group) {
  return reinterpret_cast<const GroupNote*>(p.group_notes)[group];
}

// The splits g, g + share, ... of one (row, 4 dims) into a state; CH of them are loaded before any is
// used.
template <bool COH, int CH>
__device__ __forceinline__ void join_splits(const ExtendParams& p, const Item& it, int tile_rows, int r, int c, int g, int share,
                                            float& peak, float& tot, f32x4& acc) {
  for (int s0 = g; s0 < it.splits; s0 += CH * share) {
    float x[CH];
    f32x4 v[CH];
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const int split = s0 + k * share < it.splits ? s0 + k * share : g;  // (weight 0 below)
      const u32 at = (u32)(it.slot0 + split * it.slot_step) * (u32)tile_rows + (u32)r;
      if constexpr (COH) {
        x[k] = device_load1(p.lse, 4u * at);
        v[k] = device_load4(p.parts, 4u * (at * (u32)p.dim + 4u * (u32)c));
      } else {
        x[k] = p.lse[at];
        v[k] = *reinterpret_cast<const f32x4*>(p.parts + (int64_t)at * p.dim + 4 * c);
      }
    }
    float top = peak;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const bool live = s0 + k * share < it.splits && !(x[k] <= -1.0e29f);
      top = live ? fmaxf(top, x[k]) : top;
    }
    const float keep = expf(peak - top);
    tot *= keep;
    acc *= keep;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const bool live = s0 + k * share < it.splits && !(x[k] <= -1.0e29f);
      const float w = live ? expf(x[k] - top) : 0.0f;
      tot += w;
      acc += live ? v[k] * w : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    peak = top;
  }
}

// The splits g, g + share, ... of a row's prefix into a state of 4 dims, as above.
template <int CH>
__device__ __forceinline__ void join_prefix(const SharedParams& p, const PrefixRow& x, int c, int g, int share, float& peak,
                                            float& tot, f32x4& acc) {
  for (int s0 = g; s0 < x.splits; s0 += CH * share) {
    float lse[CH];
    f32x4 v[CH];
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const int split = s0 + k * share < x.splits ? s0 + k * share : g;
      const int64_t at = (int64_t)(x.slot + split * x.step) * p.prefix_rows + x.row;
      lse[k] = p.prefix_lse[at];
      v[k] = *reinterpret_cast<const f32x4*>(p.prefix_parts + at * p.dim + 4 * c);
    }
    float top = peak;
#pragma unroll
    for (int k = 0; k < CH; ++k) top = s0 + k * share < x.splits ? fmaxf(top, lse[k]) : top;
    const float keep = expf(peak - top);
    tot *= keep;
    acc *= keep;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const float w = s0 + k * share < x.splits ? expf(lse[k] - top) : 0.0f;
      tot += w;
      acc += s0 + k * share < x.splits ? v[k] * w : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    peak = top;
  }
}

// Rows [row_from, row_to) of a split tile from its partials, by the whole workgroup. A thread holds 4
// dims of a row; where `share_rows` rows leave threads over, they share its splits (both joins of a
// short tile pass all its rows there, and so add in the same order). Weights exp(LSE - peak), empty
// splits (LSE -1e30) weigh nothing, an all-empty row is zero. COH: the partials were written by this
// launch. Uses 24 bytes of LDS a thread.
template <bool BF16, bool COH, class P>
__device__ __forceinline__ void join_rows(const P& p, const Item& it, int tile_rows, int row_from, int row_to,
                                          int share_rows, unsigned char* lds, int tid, int threads) {
  using E = Elem<BF16>;
  f32x4* const sacc = reinterpret_cast<f32x4*>(lds);
  float* const speak = reinterpret_cast<float*>(lds + threads * 16);
  float* const stot = speak + threads;
  const int d4n = p.dim / 4, pairs = (row_to - row_from) * d4n;
  const int share = share_rows * d4n < threads ? threads / (share_rows * d4n) : 1;  // threads of a (row, 4 dims) pair
  for (int base = 0; base < pairs; base += threads) {
    const int pair = share > 1 ? tid % pairs : base + tid, g = share > 1 ? tid / pairs : 0;
    const bool act = pair < pairs && g < share;
    const int r = row_from + pair / d4n, c = pair % d4n;
    float peak = kNegBig, tot = 0.0f;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    if (act) {
      if (it.splits <= 2 * share)
        join_splits<COH, 2>(p, it, tile_rows, r, c, g, share, peak, tot, acc);
      else if (it.splits <= 4 * share)
        join_splits<COH, 4>(p, it, tile_rows, r, c, g, share, peak, tot, acc);
      else
        join_splits<COH, 8>(p, it, tile_rows, r, c, g, share, peak, tot, acc);
      if constexpr (kIsSuffix<P>) {
        if (it.group >= 0)
          join_prefix<4>(p, prefix_row(p, group_note(p, it.group), it.first, it.head, it.tile * tile_rows + r), c, g,
                         share, peak, tot, acc);
      }
    }
    if (share > 1) {  // uniform
      sacc[tid] = acc;
      speak[tid] = peak;
      stot[tid] = tot;
      __syncthreads();
      if (act && g == 0) {
        float top = peak;
        for (int k = 1; k < share; ++k) top = fmaxf(top, speak[k * pairs + pair]);
        const float keep = expf(peak - top);
        acc *= keep;
        tot *= keep;
        for (int k = 1; k < share; ++k) {
          const float w = expf(speak[k * pairs + pair] - top);
          acc += sacc[k * pairs + pair] * w;
          tot += stot[k * pairs + pair] * w;
        }
      }
    }
    if (act && g == 0) {
      const float inv = 1.0f / fmaxf(tot, 1.0e-30f);
      u32x2 w;
      w.x = E::pack2(acc[0] * inv, acc[1] * inv);
      w.y = E::pack2(acc[2] * inv, acc[3] * inv);
      *reinterpret_cast<u32x2*>(static_cast<u16*>(p.out) + out_row(p, it, it.tile * tile_rows + r) + 4 * c) = w;
    }
  }
}

// ---- requests of few rows -----------------------------------------------------------------------

// dma_saddr with a non-temporal load, for keys that a call reads once: they take no place from others in
// the 256 MB cache. Ordinary / non-temporal, us: B 32, lengths 1024-4096, D 128 74.4 / 69.0, D 256
// 135 / 125; 64 requests of 8192 keys 362 / 328; one of 32768 33.4 / 31.0; small or shared pages alike (32
// requests over the same 4096 keys 56.7 / 56.8, B 4 KV 4096 19.1 / 19.7), and where several tiles read
// the same keys it goes either way (8 requests of 8192 keys, 36 / 64 / 128 rows: 68.7 / 73.8, 70.9 / 67.7,
// 112.5 / 111.3).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma_once(const void* base, u32 voff, u32 lds) {
  const uint64_t b = (uint64_t)base;
  const uint64_t ub = ((uint64_t)uniform_u32((u32)(b >> 32)) << 32) | uniform_u32((u32)b);
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1 nt"
               :
               : "v"(voff), "s"(ub), "s"(uniform_u32(lds))
               : "memory", "m0");
}
#pragma clang diagnostic pop

// The DMA of the tiles (of 32 keys, or BN) that one wave helps to fetch, tile n at key first_pos + step n, in tiles
// laid out as fwd_kernel's (C: its Cfg, of which the NWQ waves of a key group share a tile). The
// loads are inline assembly (dma_saddr, dma_flat): the compiler would wait for all of them before
// each transposing read of V; the kernels place the waits. Row offsets come from page ids that lane
// l holds for the wave's load instruction l % U of tile l / U, four such windows read at a time: a
// read in the main loop would wait for the DMA in front of it. ONCE: a request's keys are read by few
// tiles (false: by many, in loops that wait for all of the DMA anyway: ordinary loads, and one window of
// page ids, in fewer registers).
// Keys outside [lo, hi) or in pages outside the pool read zeros, and so do dims past D. Tiles with
// an instruction whose keys straddle pages are resolved key by key.
template <class C, bool ONCE = true>
struct KeyStream {
  static constexpr int U = C::INSTR_PER_WAVE;
  static constexpr int kWindow = 64 / U;  // tiles of a window
  static constexpr int kAllLive = C::RPI << 8;
  static_assert(C::BN == 32 || C::BN == 64, "a lane for every key of a tile");
  const int32_t* const table_b;
  const char* const kb;
  const char* const vb;
  const int64_t row_bytes;
  const int lane, wq, first_pos, step, my_n, lo, hi, dim;
  const u32 page, page_magic, page_shift, last_page;
  const int64_t pool_rows;
  int32_t id0 = 0, id1 = 0, id2 = 0, id3 = 0;
  // The lane's unit in the current window: pool byte offset of its first key (-1: it straddles
  // pages), and its live keys [live & 255, live >> 8).
  int64_t off = 0;
  int live = 0;

  __device__ __forceinline__ KeyStream(const ExtendParams& p, const int32_t* table, const Item& it, int lane_,
                                       int wq_, int first_pos_, int step_, int my_n_)
      : table_b(table + (int64_t)it.b * p.width),
        kb(static_cast<const char*>(p.k) + (int64_t)it.head * p.dim * 2),
        vb(static_cast<const char*>(p.v) + (int64_t)it.head * p.dim * 2),
        row_bytes((int64_t)p.heads * p.dim * 2), lane(lane_),
        wq(wq_), first_pos(first_pos_), step(step_), my_n(my_n_), lo(it.lo), hi(it.hi),
        dim(p.dim), page((u32)p.page_size), page_magic(p.page_magic), page_shift(p.page_shift),
        last_page((u32)p.width - 1u), pool_rows(p.pool_rows) {
    if (my_n > 0) read_ids(0);
  }
  __device__ __forceinline__ int unit_pos(int n) const {
    return first_pos + step * n + C::RPI * (lane % U * C::NWQ + wq);
  }
  __device__ __forceinline__ int32_t read_id(int n0) const {
    const u32 pg = div_page((u32)unit_pos(n0 + lane / U), page_magic, page_shift);
    return table_b[pg < last_page ? pg : last_page];
  }
  __device__ __forceinline__ void read_ids(int n0) {
    id0 = read_id(n0);
    if constexpr (!ONCE) return;
    id1 = read_id(n0 + kWindow);
    id2 = read_id(n0 + 2 * kWindow);
    id3 = read_id(n0 + 3 * kWindow);
  }
  // The compiler's wait for the page ids comes here.
  __device__ __forceinline__ void ids_ready() const {
    if (my_n <= 0) return;
    asm volatile("" ::"v"(id0));
    if constexpr (ONCE) asm volatile("" ::"v"(id1), "v"(id2), "v"(id3));
  }
  __device__ __forceinline__ void set_window(int n0) {
    const int w = ONCE ? n0 / kWindow % 4 : 0;
    if (w == 0 && n0 > 0) read_ids(n0);
    const int32_t a = id0, b = id1, c = id2, d = id3;  // (values: a choice of members would keep them in memory)
    const int32_t id = w == 0 ? a : w == 1 ? b : w == 2 ? c : d;
    const int n = n0 + lane / U, pos = unit_pos(n);
    const u32 pg = div_page((u32)pos, page_magic, page_shift), in_page = (u32)pos - pg * page;
    const int64_t row0 = (int64_t)id * page + in_page;
    const int from = lo > pos ? lo - pos : 0, to = hi - pos < C::RPI ? hi - pos : C::RPI;
    const bool any = n < my_n && to > from;
    const bool inside = row0 >= 0 && row0 + C::RPI <= pool_rows;
    const bool straddles = any && in_page + C::RPI > page;
    off = straddles ? -1 : any && inside ? row0 * row_bytes : 0;
    live = any && inside ? from | to << 8 : 0;
  }
  // The wave's part of the K (IS_V false) or V tile n into LDS at dst; tiles in order, K before V.
  template <bool IS_V>
  __device__ __forceinline__ void issue(const DmaLanes<C>& dl, int n, u32 dst) {
    if (!IS_V && n % kWindow == 0) set_window(n);
    const char* base = IS_V ? vb : kb;
    const int first = n % kWindow * U;
    constexpr uint64_t kUnits = (1ull << U) - 1ull;
    if ((__ballot(live != kAllLive || off < 0) >> first & kUnits) == 0 && dim == C::DPAD) {
#pragma unroll
      for (int q = 0; q < U; ++q) {
        const char* const src = base + readlane64(off, first + q);
        const u32 at = IS_V ? dl.vq(q, wq) : dl.kq(q, wq), to = dst + 1024u * (u32)(q * C::NWQ + wq);
        if constexpr (ONCE)
          dma_once(src, at, to);
        else
          dma_saddr(src, at, to);
      }
      return;
    }
    if (__ballot(off < 0) >> first & kUnits) {
      issue_keys<IS_V>(base, first_pos + step * n, dst);
      return;
    }
    const char* zero = reinterpret_cast<const char*>(kZeroChunk);
    const int lr = opaque_lane(lane) / C::CPR;
#pragma unroll
    for (int q = 0; q < U; ++q) {
      const char* const src = base + readlane64(off, first + q);
      const int keys = __builtin_amdgcn_readlane(live, first + q);
      const u32 at = IS_V ? dl.vq(q, wq) : dl.kq(q, wq);
      const bool in = lr >= (keys & 255) && lr < keys >> 8 && at - dl.row_off < 2u * (u32)dim;
      dma_flat(in ? src + at : zero, dst + 1024u * (u32)(q * C::NWQ + wq));
    }
  }
  // The same, each key through the table: lane l (mod BN) resolves key l, the load instructions fetch
  // their rows' offsets from those lanes.
  template <bool IS_V>
  __device__ __forceinline__ void issue_keys(const char* base, int pos0, u32 dst) {
    const int ln = opaque_lane(lane);
    const char* zero = reinterpret_cast<const char*>(kZeroChunk);
    const int pos = pos0 + (ln & (C::BN - 1));
    const bool in = pos >= lo && pos < hi;
    const u32 pg = in ? div_page((u32)pos, page_magic, page_shift) : 0u;
    const int64_t row = (int64_t)table_b[pg] * page + ((u32)pos - pg * page);
    const int64_t ro_own = in && row >= 0 && row < pool_rows ? row * row_bytes : -1;
#pragma unroll
    for (int q = 0; q < U; ++q) {
      const int i = q * C::NWQ + wq, r = C::RPI * i + ln / C::CPR, at = ln % C::CPR;
      const u32 rl = (u32)__builtin_amdgcn_ds_bpermute(4 * r, (int)(u32)ro_own);
      const u32 rh = (u32)__builtin_amdgcn_ds_bpermute(4 * r, (int)((uint64_t)ro_own >> 32));
      const int64_t ro = (int64_t)(((uint64_t)rh << 32) | rl);
      const int c = IS_V ? at ^ (4 * (r % C::VSW)) : at ^ (r % C::KSW);
      dma_flat(ro >= 0 && c * 8 < dim ? base + ro + c * 16 : zero, dst + 1024u * (u32)i);
    }
  }
};

// Q^T operands of the lane's row of an item's tile (row `in_tile` of it): dims 16 kk + 8 hh ..
template <class C>
__device__ __forceinline__ void load_q(const ExtendParams& p, const Item& it, int row, bool mine, int hh,
                                       u32x4 (&qf)[C::KK]) {
  const int token = row / p.group, in_group = row - token * p.group;
  const char* qp = static_cast<const char*>(p.q) + (int64_t)(it.first + token) * p.q_token +
                   (int64_t)(it.head * p.group + in_group) * p.q_head;
#pragma unroll
  for (int kk = 0; kk < C::KK; ++kk) {
    const int d = 16 * kk + 8 * hh;
    u32x4 val = {0u, 0u, 0u, 0u};
    if (mine && d < p.dim) val = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(qp + 2 * d));
    qf[kk] = val;
  }
}

// Rows that few requests' tokens fill: 32 rows to a tile, four waves that each stream their own
// 32-key blocks of the tile through LDS and meet at its end (the key layout of fwd_kernel, whose
// operand layouts and softmax these are).
//
// Each wave keeps kStages blocks of its own on the way: the K tile of block n + kStages is issued
// as soon as the scores of block n are computed, its V tile after the products of block n, and the
// waits count the half blocks issued since. One stage at head-dim tile 128 leaves room for two
// workgroups on a CU, which pays where tiles are short (B 256, lengths 75-300: 51 us, 74 with two
// stages and one workgroup) and costs nothing where they are long.
//
// The weights P of the PV product are the sum of two numbers of the input type (softmax_exp_two), so
// that an output is as exact as its own rounding: the memory bounds this kernel, and the second product
// costs 0-2% (D 128, us, one number / two: B 32 lengths 1024-4096 68.0 / 69.4, B 1 KV 32768 30.5 /
// 30.9, 8 x 8 tokens KV 2048-8192 41.9 / 42.0, 120 rows of 2048 keys 19.3 / 19.7). With one, where a
// few keys carry a row, its error was up to 1.8 times that of the output's rounding.
// Bound: B 32, lengths 1024-4096, 4.9 TB/s, by what a CU reads of the longest tile (D 256 5.4); 64
// requests of 8192 keys 6.5 TB/s; one of 32768 4.4 TB/s. One of 512 keys (Hq 8, Hkv 2, D 64) takes
// 8.4 us: a chain of dependent reads (lengths, page ids, keys) and four rounds. At D 64 a round moves
// half the bytes of D 128 through the same chain, hence the lower rate of a CU; at D 80 and 96 every
// instruction selects an address to a lane, since the tile has dims past D.
template <int DPAD>
constexpr int kStages = DPAD >= 128 ? 1 : DPAD == 64 ? 2 : 4;

// Waits until K (V) of a block has landed with `rem` further blocks of the wave to come: behind K
// are V and the halves of the next kStages - 1 blocks, behind V those and one K more.
template <class C, bool IS_V, int R = 0>
__device__ __forceinline__ void wait_half(int rem) {
  constexpr int S = kStages<C::DPAD>;
  if constexpr (R < S) {
    if (rem == R) {
      wait_vm<C::INSTR * (2 * R + (IS_V ? 0 : 1))>();
      return;
    }
    wait_half<C, IS_V, R + 1>(rem);
  } else {
    wait_vm<C::INSTR * (2 * S - 1)>();
  }
}

// LDS reads of this wave have returned: their tile may be written again.
__device__ __forceinline__ void wait_lds() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xC07F);
  asm volatile("" ::: "memory");
}

// The two numbers of a packed pair.
typedef float f32x2 __attribute__((ext_vector_type(2)));
template <bool BF16>
__device__ __forceinline__ f32x2 unpack2(u32 w) {
  if constexpr (BF16) return f32x2{__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
  const f16x2 h = __builtin_bit_cast(f16x2, w);
  return f32x2{(float)h[0], (float)h[1]};
}

// p = exp2(s * scale_log2 - m) as the sum of two numbers of the input type, hi + lo (the rest, rounded),
// operands of the PV product; returns the lane's part of the row sum.
template <class C>
__device__ __forceinline__ float softmax_exp_two(const f32x16& s, float m, float scale_log2, u32x4 (&hi)[C::KS],
                                                 u32x4 (&lo)[C::KS]) {
  using E = Elem<C::BF16>;
  float e[16], rs[4];
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    e[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[v], scale_log2, -m));
    rs[v % 4] = v < 4 ? e[v] : rs[v % 4] + e[v];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const u32 w = E::pack2(e[2 * i], e[2 * i + 1]);
    const f32x2 back = unpack2<C::BF16>(w);
    hi[i / 4][i % 4] = w;
    lo[i / 4][i % 4] = E::pack2(e[2 * i] - back[0], e[2 * i + 1] - back[1]);
  }
  return (rs[0] + rs[1]) + (rs[2] + rs[3]);
}

// The rows of an unsplit tile of a request with a prefix: the four waves' states (cm, cl, co of
// extend_tile) and the prefix's partials. Threads that rows times dims leave over share a row's partials.
template <class C>
__device__ __forceinline__ void finish_shared(const SuffixParams& p, const Item& it, const GroupNote& note, const float* cm, const float* cl,
                                              const float* co, unsigned char* lds, int tid) {
  using E = Elem<C::BF16>;
  constexpr int threads = C::THREADS;
  const int d4n = p.dim / 4, pairs = it.rows * d4n;
  const int share = pairs < threads ? threads / pairs : 1;
  for (int base = 0; base < pairs; base += threads) {
    const int pair = share > 1 ? tid % pairs : base + tid, g = share > 1 ? tid / pairs : 0;
    const bool act = pair < pairs && g < share;
    const int r = pair / d4n, c = pair % d4n;
    float peak = kNegBig, tot = 0.0f;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    if (act) {
      if (g == 0) {
        float mm = kNegBig;
#pragma unroll
        for (int k = 0; k < C::NWK; ++k) mm = fmaxf(mm, cm[k * C::ROWS_WAVE + r]);
#pragma unroll
        for (int k = 0; k < C::NWK; ++k) {
          const float wt = __builtin_amdgcn_exp2f(cm[k * C::ROWS_WAVE + r] - mm);
          tot += cl[k * C::ROWS_WAVE + r] * wt;
          acc += *reinterpret_cast<const f32x4*>(co + (k * C::ROWS_WAVE + r) * C::OSTRIDE + 4 * c) * wt;
        }
        peak = mm * kLn2;
      }
      join_prefix<8>(p, prefix_row(p, note, it.first, it.head, it.tile * C::ROWS_TILE + r), c, g, share, peak, tot, acc);
    }
    if (share > 1) {  // uniform; one pass
      f32x4* const sacc = reinterpret_cast<f32x4*>(lds);
      float* const speak = reinterpret_cast<float*>(lds + threads * 16);
      float* const stot = speak + threads;
      __syncthreads();  // the waves' states are read
      sacc[tid] = acc;
      speak[tid] = peak;
      stot[tid] = tot;
      __syncthreads();
      if (act && g == 0) {
        float top = peak;
        for (int k = 1; k < share; ++k) top = fmaxf(top, speak[k * pairs + pair]);
        const float keep = expf(peak - top);
        acc *= keep;
        tot *= keep;
        for (int k = 1; k < share; ++k) {
          const float w = expf(speak[k * pairs + pair] - top);
          acc += sacc[k * pairs + pair] * w;
          tot += stot[k * pairs + pair] * w;
        }
      }
    }
    if (act && g == 0) {
      const float inv = 1.0f / fmaxf(tot, 1.0e-30f);
      u32x2 w;
      w.x = E::pack2(acc[0] * inv, acc[1] * inv);
      w.y = E::pack2(acc[2] * inv, acc[3] * inv);
      *reinterpret_cast<u32x2*>(static_cast<u16*>(p.out) + out_row(p, it, it.tile * C::ROWS_TILE + r) + 4 * c) = w;
    }
  }
}

template <class C, class P>
__device__ __forceinline__ void extend_tile(const P& p, const int32_t* table, const Item& it,
                                            unsigned char* smem, int tid, bool fused) {
  // (Opaque copies: what derives from the lane is computed here and at the end, not held across the
  // caller's loop.)
  tid = opaque_lane(tid);
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int il = lane & 31, hh = lane >> 5;
  const Lanes<C> ln(lane);
  GroupNote note = {};
  if constexpr (kIsSuffix<P>)
    if (it.group >= 0) note = group_note(p, it.group);
  constexpr int S = kStages<C::DPAD>;
  unsigned char* const stages = smem + wave * S * C::STAGE_BYTES;
  const u32 stages_lds = lds_address(stages);

  // This wave's blocks: blk_begin + wave, + 4, ...
  constexpr int kStep = C::NWK * C::BN;
  const int cnt = it.blk_end - it.blk_begin;
  const int my_n = cnt > wave ? (cnt - wave + C::NWK - 1) / C::NWK : 0;
  const int first_pos = (it.blk_begin + wave) * C::BN;
  KeyStream<C> keys(p, table, it, lane, 0, first_pos, kStep, my_n);
  const DmaLanes<C> dl(lane, 0, keys.row_bytes);
  auto issue_k = [&](int n) { keys.template issue<false>(dl, n, stages_lds + (u32)(n % S * C::STAGE_BYTES)); };
  auto issue_v = [&](int n) {
    keys.template issue<true>(dl, n, stages_lds + (u32)(n % S * C::STAGE_BYTES) + (u32)C::TILE_BYTES);
  };

  const int row = it.tile * C::ROWS_TILE + il;
  const int token = row / p.group;
  u32x4 qf[C::KK];
  load_q<C>(p, it, row, il < it.rows, hh, qf);
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

  // (The compiler's waits for page ids and Q, older than the DMA, come here and not in the loop.)
  keys.ids_ready();
  for (int n = 0; n < S && n < my_n; ++n) {
    issue_k(n);
    issue_v(n);
  }
#pragma unroll
  for (int kk = 0; kk < C::KK; ++kk) asm volatile("" ::"v"(qf[kk]));
  for (int n = 0; n < my_n; ++n) {
    const int pos0 = first_pos + kStep * n;
    const unsigned char* stage = stages + n % S * C::STAGE_BYTES;
    const int rem = my_n - 1 - n;
    // One or two waves to a SIMD hide little of a chain of LDS reads and products. So all operands of
    // a product are read at once (there are registers for them), the scores come in two chains, K's
    // next tile is issued while they run, and V is read under the softmax.
    u32x4 ka[C::KK], va[C::KS * C::DT], pf[C::KS], pl[C::KS];
    f32x16 s[1], t;
    wait_half<C, false>(rem);
    asm volatile("" ::: "memory");
#pragma unroll
    for (int kk = 0; kk < C::KK; ++kk) ka[kk] = read_k<C>(stage, ln, 0, kk);
    wait_lds();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int v = 0; v < 16; ++v) s[0][v] = t[v] = 0.0f;
#pragma unroll
    for (int kk = 0; kk < C::KK; kk += 2) {
      s[0] = Elem<C::BF16>::mma(ka[kk], qf[kk], s[0]);
      t = Elem<C::BF16>::mma(ka[kk + 1], qf[kk + 1], t);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (rem >= S) issue_k(n + S);
    wait_half<C, true>(rem);
    asm volatile("" ::: "memory");
#pragma unroll
    for (int k2 = 0; k2 < C::KS; ++k2)
#pragma unroll
      for (int dt = 0; dt < C::DT; ++dt) va[k2 * C::DT + dt] = read_vt<C>(stage + C::TILE_BYTES, ln, dt, k2);
    __builtin_amdgcn_sched_barrier(0);
    s[0] += t;
    if (pos0 + C::BN > hi_min || pos0 < lo_max) mask_seen<C>(s, pos0, seen, hh);
    float sum = softmax_exp_two<C>(s[0], m, p.scale_log2, pf, pl);
    if (__ballot(!(sum <= kSoftmaxSumBound))) {
      const float top = fmaxf(m, row_max<C>(s, p.scale_log2));
      const float keep = __builtin_amdgcn_exp2f(m - top);
      l *= keep;
#pragma unroll
      for (int dt = 0; dt < C::DT; ++dt) o[dt] *= keep;
      m = top;
      sum = softmax_exp_two<C>(s[0], m, p.scale_log2, pf, pl);
    }
    l += sum;
    wait_lds();
    if (rem >= S) issue_v(n + S);
#pragma unroll
    for (int k2 = 0; k2 < C::KS; ++k2) {
#pragma unroll
      for (int dt = 0; dt < C::DT; ++dt)
        o[dt] = Elem<C::BF16>::mma(va[k2 * C::DT + dt], pf[k2], o[dt]);
#pragma unroll
      for (int dt = 0; dt < C::DT; ++dt)
        o[dt] = Elem<C::BF16>::mma(va[k2 * C::DT + dt], pl[k2], o[dt]);
    }
  }

  // The waves' states of the same rows, through LDS.
  __syncthreads();
  tid = opaque_lane(tid);
  const int cil = tid & 31, chh = (tid & 63) >> 5;
  float* cm = reinterpret_cast<float*>(smem);
  float* cl = cm + C::NWK * C::ROWS_WAVE;
  float* co = cl + C::NWK * C::ROWS_WAVE;
  const float tot = pair_sum(l);
  if (chh == 0) {
    cm[wave * C::ROWS_WAVE + cil] = m;
    cl[wave * C::ROWS_WAVE + cil] = tot;
  }
  if (cil < it.rows) {
#pragma unroll
    for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
      for (int gq = 0; gq < 4; ++gq) {
        f32x4 val = {o[dt][4 * gq], o[dt][4 * gq + 1], o[dt][4 * gq + 2], o[dt][4 * gq + 3]};
        *reinterpret_cast<f32x4*>(co + (wave * C::ROWS_WAVE + cil) * C::OSTRIDE + 32 * dt + 8 * gq +
                                  4 * chh) = val;
      }
  }
  __syncthreads();
  using E = Elem<C::BF16>;
  if constexpr (kIsSuffix<P>) {
    if (it.splits == 1 && it.group >= 0) {
      finish_shared<C>(p, it, note, cm, cl, co, smem, tid);
      return;
    }
  }
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
    if (it.splits == 1 && !kIsPrefix<P>) {
      u32x2 w;
      w.x = E::pack2(acc[0] * inv, acc[1] * inv);
      w.y = E::pack2(acc[2] * inv, acc[3] * inv);
      *reinterpret_cast<u32x2*>(static_cast<u16*>(p.out) +
                                out_row(p, it, it.tile * C::ROWS_TILE + r) + d0) = w;
      continue;
    }
    const u32 at = (u32)it.slot * C::ROWS_TILE + (u32)r;
    acc *= inv;
    if (fused) {
      device_store4(p.parts, 4u * (at * (u32)p.dim + (u32)d0), acc);
      if (d0 == 0) device_store1(p.lse, 4u * at, part_lse(mm, t2));
    } else {
      *reinterpret_cast<f32x4*>(p.parts + (int64_t)at * p.dim + d0) = acc;
      if (d0 == 0) p.lse[at] = part_lse(mm, t2);
    }
  }
}

// One item a program. With counters the program that writes the last split of a tile joins it (and
// sets the tile's counter, that of its first item, back to zero); else a second launch does.
template <class C, class P>
__global__ __launch_bounds__(C::THREADS, C::DPAD == 256 ? 1 : 2) void extend_rows_kernel(
    P p, const int32_t* __restrict__ table, const int32_t* __restrict__ lengths,
    const int32_t* __restrict__ cu) {
  constexpr int kBytes = CMax<C::NWK * kStages<C::DPAD> * C::STAGE_BYTES, C::COMB_BYTES>::value;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[kBytes];
  const int tid = threadIdx.x;
  Item it;
  const bool found = find_item<ShortTiling>(p, lengths, cu, (int)blockIdx.x, tid & 63, it);
  write_note(p, it, found);
  if (!found) return;
  const bool fused = p.counters != nullptr && !kIsPrefix<P>;
  extend_tile<C>(p, table, it, smem, tid, fused);
  if constexpr (kIsPrefix<P>) return;
  if (it.splits == 1 || !fused) return;
  wait_vm<0>();     // this wave's partials are complete at the device
  __syncthreads();  // ... and every wave's
  int* const flag = reinterpret_cast<int*>(smem);
  int32_t* const counter = p.counters + (int64_t)it.slot0 * kArrivalStride;
  if (tid == 0)
    *flag = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == it.splits - 1;
  __syncthreads();
  const bool last = *flag != 0;
  __syncthreads();  // LDS is written again
  if (!last) return;
  join_rows<C::BF16, true>(p, it, C::ROWS_TILE, 0, it.rows, it.rows, smem, tid, C::THREADS);
  if (tid == 0) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The joins that the kernels leave: blockIdx.x items of the rows kernel, then of the long one. The
// programs of a tile's splits share its rows, kJoinParts of them (blockIdx.y) to a split of a long
// tile: few programs, since one takes 5 ns to dispatch.
constexpr int kJoinParts = 4;
template <bool BF16, class P>
__global__ __launch_bounds__(kMergeThreads) void extend_join_kernel(P rows, P longs, int rows_items) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[kMergeThreads * 24];
  auto join = [&](const P& p, int w, int tile_rows, int per_split, bool whole) {
    const JoinNote note = reinterpret_cast<const JoinNote*>(p.notes)[w];
    if (note.splits < 2) return;
    Item it;
    it.first = note.first;
    it.tile = note.tile;
    it.head = note.head;
    it.splits = note.splits;
    it.slot0 = w - note.split * p.heads;
    it.slot_step = p.heads;
    it.group = note.group;
    const int parts = note.splits * per_split, part = note.split * per_split + (int)blockIdx.y;
    const int from = note.rows * part / parts, to = note.rows * (part + 1) / parts;
    if (from < to)
      join_rows<BF16, false>(p, it, tile_rows, from, to, whole ? note.rows : to - from, lds, threadIdx.x, kMergeThreads);
  };
  if ((int)blockIdx.x >= rows_items)
    join(longs, (int)blockIdx.x - rows_items, longs.dim > 128 ? WideTiling::ROWS : LongTiling::ROWS, kJoinParts, false);
  else if (blockIdx.y == 0)
    join(rows, (int)blockIdx.x, ShortTiling::ROWS, 1, true);
}

template <bool BF16, int DPAD, class P>
hipError_t launch_extend_rows(const P& p, int grid, hipStream_t stream) {
  using C = Cfg<BF16, DPAD, kLayoutKey, DPAD == 128 ? 1 : 0>;
  extend_rows_kernel<C, P><<<dim3(grid), dim3(C::THREADS), 0, stream>>>(p, p.table, p.lengths, p.cu);
  return hipGetLastError();
}

}  // namespace fgw_kv
