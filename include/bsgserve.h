/*
 * bsgserve.h — C ABI of the serving operators beside the block-sparse GEMM on the MI355X (gfx950):
 * a paged cache of keys and values held in 8 bits, the attention that reads it, the bookkeeping
 * of its pages, and the log probabilities of tokens.  They have no counterpart in the reference,
 * whose decode drivers leave attention and cache to the model's own library.
 *
 * Conventions as in bsgemm.h: device pointers, `stream` a hipStream_t as void*, no allocation and
 * no synchronisation, arguments checked on the host before any HIP call, BSG_OK or a BSG_ERR_*
 * code with bsg_last_error().  Values that only the device knows (lengths, page ids, slots, token
 * offsets) are checked there: what lies outside its range is skipped, never followed.
 *
 * The cache of one layer.  A page holds page_size tokens of every head.  pages is
 * [num_pages][n_heads][2][page_size][head_dim] in e4m3 (OCP, no infinities), keys then values;
 * scales is fp32 [num_pages][n_heads][2], one power of two for the keys and one for the values of
 * each page and head: a cached number is its e4m3 value times its scale.  Inside
 * [page_size][head_dim] lie tiles of 16 tokens x 64 channels, 1 KiB each, in the lane order of a
 * 16-byte-per-lane load:
 *   keys   byte 256 g + 16 t + e       = token t, channel 16 g + e            (e < 16)
 *   values byte 256 g + 16 l + 4 i + t = token 4 g + t, channel 16 i + l      (t < 4, i < 4)
 * tile (16-token block a, 64-channel block c) at byte 16 head_dim a + 1024 c.  Either tile is then
 * the A operand of v_mfma_f32_16x16x32 after conversion, with no shuffle and no LDS.
 * page_table[slot][j] names the page of tokens j page_size .. of a sequence, -1 none.
 */
#ifndef BSGSERVE_H
#define BSGSERVE_H

#include <stdint.h>

#include "bsgemm.h"

#ifdef __cplusplus
extern "C" {
#endif

#define BSG_F32 2                     /* logits only */
#define BSG_KV_SCALE_MIN_EXP (-40)    /* scales lie in [2^-40, 2^80] */
#define BSG_KV_SCALE_MAX_EXP 80
#define BSG_KV_MAX_TOKENS (1 << 30)   /* max_pages x page_size of a table */
#define BSG_PAGES_MAX_ROWS 1024       /* slots of one fork, extend or free call */
#define BSG_LOGPROBS_MAX_K 64

typedef struct bsg_kv_cache {
  void* pages;               /* one layer; 16-byte aligned */
  float* scales;             /* 8-byte aligned */
  int64_t num_pages;         /* < 2^31 */
  int32_t n_heads;
  int32_t page_size;         /* 16, 32, 64 or 128 */
  int32_t head_dim;          /* 64 or 128 */
  int32_t num_slots;         /* rows of page_table, entries of lengths */
  int32_t max_pages;         /* columns of page_table; max_pages x page_size <= BSG_KV_MAX_TOKENS */
  int64_t table_stride;      /* elements between its rows, >= max_pages */
  const int32_t* page_table;
  const int32_t* lengths;    /* tokens of each slot, the new ones of a call among them */
} bsg_kv_cache;

/* Write the new keys and values of a batch into the cache.
 *   k, v     : [tokens][n_heads][head_dim] fp16/bf16, strides in elements (channels contiguous)
 *   slots    : the slot of each of `rows` sequences, or NULL for 0 .. rows-1; others are skipped
 *   cu       : rows + 1 token offsets, or NULL when every sequence has max_new tokens
 *              (tokens == rows * max_new)
 *   max_new  : at least the most tokens of one sequence (later ones are neither written nor weighed)
 * Row b's new tokens are the last cu[b+1] - cu[b] of its lengths[slot].  Per page, head and K/V:
 * a = the largest finite magnitude among the new tokens, scale = the least power of two >= a / 448,
 * and no less than the page's scale if it holds earlier tokens, which are rounded again when the scale grows
 * (exact but for values that become subnormal).  x / scale is rounded to nearest even; +-448 where
 * it is infinite, NaN where it is NaN.  The written pages must belong to one sequence each. */
int bsg_kv_append(const void* k, int64_t k_stride_t, int64_t k_stride_h, const void* v, int64_t v_stride_t,
                  int64_t v_stride_h, int64_t tokens, const bsg_kv_cache* cache, const int32_t* slots, int32_t rows,
                  const int32_t* cu, int32_t max_new, int dtype, void* stream);

/* Attention of the newest tokens of every sequence over its cached tokens (their own among them,
 * appended before): new token i of n sees the first length - n + i + 1 tokens,
 *   out = softmax(sm_scale * q . k) v      lse = log of the softmax's sum (natural, fp32)
 *   q, out   : [tokens][q_heads][head_dim], q_heads a multiple of n_heads; query head h reads
 *              cached head h / (q_heads / n_heads); rows 16-byte (q) and 8-byte (out) aligned
 *   lse      : [tokens][q_heads], or NULL
 *   sm_scale : finite, as log2(e) times it
 *   max_len  : at least the longest sequence, for the split over the long axis only (any length
 *              is computed rightly)
 * A token that sees nothing gives zeros and -inf, as do the tokens of a sequence whose slot is out of
 * range; rows of q that cu gives to no sequence are not computed.  Tokens on a page id out of range are not seen.  Products of 16-bit operands (keys and
 * values converted exactly, probabilities in fp16 after a shift by 2^13), sums, maxima and
 * exponentials in 32 bits.  Workspace: 16-byte aligned, its first BSG_KV_COUNTER_BYTES zero before
 * the first use and left zero; calls that may overlap must not share one. */
#define BSG_KV_COUNTER_BYTES 65536
int64_t bsg_kv_attention_workspace_bytes(const bsg_kv_cache* cache, int32_t rows, int32_t q_heads, int32_t max_new,
                                         int64_t max_len, int32_t cu_count);
int bsg_kv_attention(const void* q, int64_t q_stride_t, int64_t q_stride_h, int64_t tokens, int32_t q_heads,
                     const bsg_kv_cache* cache, const int32_t* slots, int32_t rows, const int32_t* cu,
                     int32_t max_new, int64_t max_len, float sm_scale, void* out, int64_t o_stride_t,
                     int64_t o_stride_h, float* lse, int dtype, void* ws, int64_t ws_bytes, int32_t cu_count,
                     void* stream);

/* The pool of pages behind the layers of a cache: pages [layers][num_pages][page_bytes] and scales
 * [layers][num_pages][page_scales], both contiguous.  refcounts[p] is the number of page_table
 * entries that name page p; 0 = free. */
typedef struct bsg_page_pool {
  void* pages;            /* 16-byte aligned; NULL where a call moves no data */
  float* scales;
  int64_t layers;
  int64_t num_pages;      /* < 2^31 */
  int64_t page_bytes;     /* of one layer, a multiple of 16 */
  int64_t page_scales;    /* floats of one layer's page */
  int32_t page_size;
  int32_t num_slots;
  int32_t max_pages;      /* as in bsg_kv_cache */
  int64_t table_stride;
  int32_t* page_table;
  int32_t* lengths;
  int32_t* refcounts;
} bsg_page_pool;

/* Copy pages src[i] -> dst[i], i < n, in every layer, with their scales.  Pairs with an id out of
 * range are skipped.  A page may not be written twice, nor written and read, in one call. */
int bsg_pages_copy(const bsg_page_pool* pool, const int32_t* src, const int32_t* dst, int32_t n, void* stream);

/* Sequences go on from others: slot children[i] takes the pages and length of slot parents[i], all
 * at once (a slot may be both), sharing the pages; what it held before is released.  Pairs with a
 * slot out of range are skipped; of pairs with the same child the last one counts.  n <=
 * BSG_PAGES_MAX_ROWS. */
int bsg_pages_fork(const bsg_page_pool* pool, const int32_t* parents, const int32_t* children, int32_t n,
                   void* stream);

/* Room for new_tokens[i] more tokens of slot slots[i] (NULL: slot i): lengths grow, the pages they
 * need are taken from the free ones, lowest id first, in the order of the rows, and a last page
 * that other slots read as well is replaced by a copy before it is written to (the last of its
 * readers in the call keeps it).  served[i] = 1, or 0 where nothing was changed: the slot is out
 * of range, its table row is too short, or the free pages do not reach: rows are served in order
 * until the first that they do not reach; of the later ones only those that need no page and write
 * to no shared one are.  Slots must be distinct.  n <= BSG_PAGES_MAX_ROWS.
 * Workspace: bsg_pages_workspace_bytes(num_pages), no initialisation.  The call is two launches, the
 * first of which leaves the second its plan there: nothing else may write to it on the stream in
 * between, so threads that share a stream need one each. */
int64_t bsg_pages_workspace_bytes(int64_t num_pages);
int bsg_pages_extend(const bsg_page_pool* pool, const int32_t* slots, const int32_t* new_tokens, int32_t n,
                     int32_t* served, void* ws, int64_t ws_bytes, void* stream);

/* Release every page of the given slots; their rows become -1 and their lengths 0.  Slots out of
 * range are skipped, one that is named twice is released once.  n <= BSG_PAGES_MAX_ROWS. */
int bsg_pages_free(const bsg_page_pool* pool, const int32_t* slots, int32_t n, void* stream);

/* Make the pool dense: the live pages past the first `live` ids move, in order, to the free ones
 * before, with their counts, and every page_table entry follows.  counts[0] = live pages,
 * counts[1] = moved ones.  Workspace as bsg_pages_extend. */
int bsg_pages_compact(const bsg_page_pool* pool, int32_t* counts, void* ws, int64_t ws_bytes, void* stream);

/* Log probabilities of given tokens under rows of logits.
 *   logits    : [rows][vocab], row stride in elements, fp16, bf16 or fp32
 *   tokens    : int32 [rows]; a token out of range gives NaN
 *   logprob   : fp32 [rows]       logits[r, tokens[r]] - lse_r
 *   entropy   : fp32 [rows]       lse_r - sum p x, in nats
 *   top_ids   : int32 [rows][k], top_logprobs: fp32 [rows][k]: the k <= BSG_LOGPROBS_MAX_K likeliest
 *               tokens, by (logit desc, id asc); -0 equals +0 and NaN ranks above every number
 * Rows of nothing but -inf give logprob -inf and entropy 0; a NaN in a row makes every number of the
 * row NaN, as does a +inf but for its ids.  Sums in 32 bits.  The aligned 16-byte granules that a
 * row begins and ends in are read whole.  Workspace as bsg_kv_attention: BSG_KV_COUNTER_BYTES of counters, zero before the first use and left zero. */
int64_t bsg_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int32_t k, int dtype, int32_t cu_count);
int bsg_token_logprobs(const void* logits, int64_t row_stride, int64_t rows, int64_t vocab, const int32_t* tokens,
                       int32_t k, float* logprob, float* entropy, int32_t* top_ids, float* top_logprobs, int dtype,
                       void* ws, int64_t ws_bytes, int32_t cu_count, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* BSGSERVE_H */
