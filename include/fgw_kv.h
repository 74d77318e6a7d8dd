/*
 * fgw_kv.h -- C ABI of the operators around the paged K/V cache of fgw_mha.h, MI355X (gfx950).
 *
 * The cache's writer, its reader for grouped heads, and the moves of its pages:
 *   fgw_rotary_apply   rotary positions of [T, H, D] rows (and their inverse)
 *   fgw_kv_append      new tokens into the pages, Q and K rotated on the way
 *   fgw_kv_extend      attention of packed ragged new tokens over the pages, grouped K/V heads
 *   fgw_pages_*        fork, free, reserve, compact and copy pages; books on the device
 * None has a counterpart in the reference, which reads a cache that its caller has written.
 *
 * Shared conventions (those of fgw_mha.h): pool rows K, V [N, Hkv, D] contiguous, N = pages *
 * page_size; block table [B, W] int32; cache lengths [B] int32. A page id outside the pool reads
 * as zeros and is not written. New tokens are packed: request b has the rows
 * [cu[b], cu[b + 1]) of Q, K, V (cu [B + 1] int32, cu[0] = 0, never falling), and its cache length
 * counts them: its row cu[b] + j has the cache position len_b - n_b + j, n_b = cu[b + 1] - cu[b].
 * Lengths lie in [0, W * page_size], where fgw_pages_reserve keeps them. Of others fgw_kv_append
 * writes the tokens whose position has a place, while fgw_kv_extend takes the nearer end for the
 * length, and so sees other positions than those written.
 * Rows at and behind cu[B] are neither read nor written. What a call writes shares no memory with
 * what it reads, except where a rotated output may be the input itself.
 *
 * All functions return 0 or a negative fgw_mha_status; the message of the calling thread's last
 * failure is in fgw_kv_last_error(). Nothing allocates, frees or synchronises; launches are
 * asynchronous on the given stream, which belongs to the current device. Reentrant.
 */
#ifndef FGW_KV_H_
#define FGW_KV_H_

#include <stdint.h>

#include <hip/hip_runtime_api.h>

#include "fgw_mha.h"

#ifdef __cplusplus
extern "C" {
#endif

#define FGW_KV_ABI_VERSION 1

typedef enum { FGW_KV_FLOAT16 = 0, FGW_KV_BFLOAT16 = 1, FGW_KV_FLOAT32 = 2 } fgw_kv_dtype;

int fgw_kv_abi_version(void);
const char* fgw_kv_last_error(void);

/* Rotary positions: pair i of a row at position p turns by turns[i] * p * 2^-64 of a full turn,
 * taken modulo a turn in integers, so no position is too far:
 *   a' = scale (a cos t - b sin t),  b' = scale (b cos t + a sin t).
 * The pairs of the first `dim` dims are (i, i + dim / 2), or (2 i, 2 i + 1) when interleaved;
 * later dims are copied. inverse: t -> -t (the transpose of the forward, its gradient). */
typedef struct {
  const uint64_t* turns; /* [dim / 2], device; NULL: nothing is rotated (fgw_kv_append only) */
  int32_t dim;           /* rotated dims, a multiple of 16, at most the head dim */
  int32_t interleaved;
  int32_t inverse;
  float scale;
} fgw_kv_rotary;

/* Rows [tokens, heads, dim] with element strides; the last dim is contiguous. Pointers 16-byte
 * aligned, strides multiples of 16 bytes. */
typedef struct {
  const void* data;
  int64_t token_stride, head_stride;
} fgw_kv_rows;

typedef struct {
  fgw_kv_rows x;
  fgw_kv_rows out; /* may be x itself (then the dims past rotary.dim are left) */
  const void* positions; /* [tokens] */
  int32_t positions64;   /* 1: int64, 0: int32 */
  int32_t tokens, heads, dim, dtype; /* fgw_kv_dtype */
  fgw_kv_rotary rotary;
} fgw_rotary_args;

int fgw_rotary_apply(const fgw_rotary_args* args, hipStream_t stream);

typedef struct {
  fgw_kv_rows q, k, v, q_out;
  void* k_cache;
  void* v_cache;
  const int32_t* block_table;
  const int32_t* cache_seqlens;
  const int32_t* cu_seqlens;
  const void* positions; /* rotary positions [tokens], or NULL: the cache positions */
  int32_t positions64;
  int64_t pool_rows;
  int32_t tokens, batch, heads, kv_heads, dim, width, page_size;
  int32_t dtype; /* FGW_KV_FLOAT16 or FGW_KV_BFLOAT16 */
  fgw_kv_rotary rotary;
} fgw_kv_append_args;

/* Writes q_out (which may be q itself) = rotated q, and each new token's rotated K and its V to the pool row
 * table[b, pos / page] * page + pos % page. Tokens whose position lies outside [0, W * page), or
 * whose page id lies outside the pool, are not written to the pool. */
int fgw_kv_append(const fgw_kv_append_args* args, hipStream_t stream);

/* Attention over the pages with grouped heads: query head h reads K/V head h / (heads / kv_heads).
 * Row cu[b] + j sees the keys [0, len_b) (causal 0), or, with its position pos = len_b - n_b + j,
 * (pos - window, pos] of them (window 0: [0, pos]). Rows that see nothing are zero. */
typedef struct {
  fgw_kv_rows q;
  void* out; /* [tokens, heads, dim] contiguous */
  const void* k_cache;
  const void* v_cache;
  const int32_t* block_table;
  const int32_t* cache_seqlens;
  const int32_t* cu_seqlens;
  float* workspace; /* the floats of fgw_kv_extend_workspace, or NULL if that is 0 */
  int32_t* counters; /* NULL (parts of split tiles are joined by a second launch), or the counters of
                        fgw_kv_extend_workspace, all zero: the last program of a tile joins it and
                        leaves its counter at zero. Calls that may overlap need their own. */
  int64_t pool_rows;
  int32_t tokens, batch, heads, kv_heads, dim, width, page_size;
  int32_t max_new;  /* no request has more new tokens than this (more are not computed) */
  int32_t causal, window;
  int32_t dtype;    /* FGW_KV_FLOAT16 or FGW_KV_BFLOAT16 */
  int32_t num_cus;  /* compute units to fill (above 256: 256) */
  float scale;      /* of the scores */
} fgw_kv_extend_args;

/* fp32 elements of workspace and int32 counters that a call with these sizes can use (pointers are
 * not read; 0 counters: none of its joins is fused); pure host function. */
int fgw_kv_extend_workspace(const fgw_kv_extend_args* args, int64_t* floats, int64_t* counters);
int fgw_kv_extend(const fgw_kv_extend_args* args, hipStream_t stream);

/* Books of the pages, on the device: refs [pages] int32 holders of each page (0: free), table
 * [rows, width] int32, lens [rows] int32. Row r holds the pages table[r, 0 .. ceil(lens[r] /
 * page_size)). Pages are handed out lowest id first, to rows (pairs) in order, so the books are
 * the same on every run. */
typedef struct {
  int32_t* refs;
  int32_t* table;
  int32_t* lens;
  int32_t pages, rows, width, page_size;
} fgw_pages_books;

/* Pools whose pages move together: pool i holds page p at data[i] + p * page_bytes[i] (multiples
 * of 16). */
typedef struct {
  void* const* data;
  const int64_t* page_bytes;
  int32_t count;
} fgw_pages_pools;

/* int32 elements of the workspace of a call over `pages` pages and `entries` rows or pairs. */
int64_t fgw_pages_workspace(int32_t pages, int32_t entries);

/* Row r grows by counts[r] tokens: lens[r] += counts[r], and the pages that this needs are taken.
 * A row that does not fit the table (or has counts[r] < 0) stays as it is, and so does one whose
 * pages, with those of the rows before it, are more than the free ones.
 * status [2]: rows refused for want of pages, rows refused for their counts. */
int fgw_pages_reserve(const fgw_pages_books* books, const int32_t* counts, int32_t* status,
                      int32_t* workspace, hipStream_t stream);

/* Row children[i] becomes a copy of row parents[i]: the whole pages are shared, a partly filled
 * last page is copied in every pool to a fresh page. Pair i is refused when a row is out of range,
 * the child holds tokens or is a parent or an earlier pair's child (status[1]), or no page is left
 * for it (status[0]). */
int fgw_pages_fork(const fgw_pages_books* books, const fgw_pages_pools* pools,
                   const int32_t* parents, const int32_t* children, int32_t pairs, int32_t* status,
                   int32_t* workspace, hipStream_t stream);

/* The rows give their pages back: lens 0, table entries -1. Rows out of range, empty or listed
 * before are left. */
int fgw_pages_free(const fgw_pages_books* books, const int32_t* rows, int32_t count,
                   hipStream_t stream);

/* Moves the live pages to the ids below their number, L: the i-th live page from L on goes to the
 * i-th free one below L, in every pool; tables and refs follow. moved [1]: pages moved. */
int fgw_pages_compact(const fgw_pages_books* books, const fgw_pages_pools* pools, int32_t* moved,
                      int32_t* workspace, hipStream_t stream);

/* Copies page src[i] to page dst[i] in every pool; pairs with an id outside [0, pages) are
 * skipped. No page may be a destination twice, or a destination and a source. */
int fgw_pages_copy(const fgw_pages_pools* pools, int32_t pages, const int32_t* src,
                   const int32_t* dst, int32_t count, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* FGW_KV_H_ */
