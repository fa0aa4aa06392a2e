/*
 * bsgdraft.h — C ABI of the operators of a step that drafts tokens and verifies them over the 8-bit
 * paged cache of bsgserve.h: queries and keys normed and rotated on their way into it, attention of a
 * tree of drafts, their verification, and what stays of them in the cache.  They have no counterpart in
 * the reference, which decodes one token at a time.
 *
 * Conventions as in bsgserve.h.  A tree is the newest tokens of a sequence, its nodes, of which
 * parents[t] names the parent of token t by its place among them; what names no earlier node of the
 * sequence (-1) makes a node a root.  At most BSG_TREE_NODES nodes of a sequence.
 */
#ifndef BSGDRAFT_H
#define BSGDRAFT_H

#include <stdint.h>

#include "bsgserve.h"

#ifdef __cplusplus
extern "C" {
#endif

#define BSG_TREE_NODES 64

/* How queries and keys are turned.  Of a head's channels the first `dims` are rotated by the angles of
 * the token's position, in pairs (i, i + dims / 2), or with `interleaved` (2 i, 2 i + 1):
 *   (a, b) -> (a cos - b sin, a sin + b cos),  cos and sin the position's i-th. */
typedef struct bsg_rotary {
  const float* cos;            /* [positions][dims / 2], rows 16-byte aligned */
  const float* sin;            /* the same */
  int64_t stride;              /* elements between the rows of either */
  int32_t positions;
  int32_t dims;                /* 16, 32, 64 or 128, at most head_dim */
  int32_t interleaved;
  float eps;
  const void* q_norm;          /* [head_dim] in the call's type, 16-byte aligned, or NULL: */
  const void* k_norm;          /*   before the rotation x * rsqrt(mean(x^2) + eps) * norm, for each head */
  const int32_t* token_positions; /* the position of each token, or NULL: */
  const int32_t* parents;      /*   the tree's first place plus the node's depth in it, or NULL: */
} bsg_rotary;                  /*   the token's place in its sequence */

/* bsg_kv_append of keys that are normed and rotated on the way, with the queries of the same tokens:
 *   q, out   : [tokens][q_heads][head_dim], rows 16-byte aligned; out may be q
 * Everything between the inputs and the one rounding of q, k and v is in 32 bits; scales and rounding as
 * bsg_kv_append of those 32-bit numbers.  A position outside [0, positions) makes the rotated channels NaN.
 * Queries of a sequence whose slot is out of range, of tokens past max_new, and rows of q that cu gives
 * to no sequence are left as they are in out. */
int bsg_kv_append_rotated(const void* q, int64_t q_stride_t, int64_t q_stride_h, int32_t q_heads, void* out,
                          int64_t o_stride_t, int64_t o_stride_h, const void* k, int64_t k_stride_t, int64_t k_stride_h,
                          const void* v, int64_t v_stride_t, int64_t v_stride_h, int64_t tokens,
                          const bsg_rotary* rotary, const bsg_kv_cache* cache, const int32_t* slots, int32_t rows,
                          const int32_t* cu, int32_t max_new, int dtype, void* stream);

/* bsg_kv_attention of a tree: node i of a sequence's n new tokens sees its first length - n tokens,
 * its own ancestors and itself.  max_new <= BSG_TREE_NODES; everything else as there. */
int64_t bsg_kv_tree_attention_workspace_bytes(const bsg_kv_cache* cache, int32_t rows, int32_t q_heads, int32_t max_new,
                                              int64_t max_len, int32_t cu_count);
int bsg_kv_tree_attention(const void* q, int64_t q_stride_t, int64_t q_stride_h, int64_t tokens, int32_t q_heads,
                          const int32_t* parents, const bsg_kv_cache* cache, const int32_t* slots, int32_t rows,
                          const int32_t* cu, int32_t max_new, int64_t max_len, float sm_scale, void* out,
                          int64_t o_stride_t, int64_t o_stride_h, float* lse, int dtype, void* ws, int64_t ws_bytes,
                          int32_t cu_count, void* stream);

/* Which drafted tokens a target model accepts, and the token that follows them, from given random
 * numbers.  Per sequence, nodes 0 .. n-1 with n = cu[b+1] - cu[b] (max_new where cu is NULL, later ones
 * are not looked at): node 0 is accepted, then the children of the last accepted node in the order of
 * their places, until one is accepted, and so on; the first node none of whose children is ends the path.
 * With p the probabilities softmax(logits / temperature) of the last accepted node's row, x the child's
 * token, u its number:
 *   without draft_logits   accepted if u (1 - r) < p(x), r the sum of p over its rejected siblings' tokens
 *                          (one of the same token is rejected); the new token is drawn from what is left of p
 *   with draft_logits      (chains: parents NULL) q = softmax(draft_logits / temperature) of the same row;
 *                          accepted if u q(x) < p(x); after a rejection the new token is drawn from
 *                          max(p - q, 0), otherwise from p
 *   temperature <= 0       accepted if x is the likeliest token (the first of equal ones), which is also the new one
 * where nothing is left, from p.  Drawn: the first token whose running sum exceeds uniforms[node 0] times the whole.
 * Decisions are those of 64-bit weights and sums (32-bit ones only decide what they cannot have wrong), so that the answer is
 * the definition's but for numbers within some 2^-40 of a border.
 *   logits, draft_logits : [tokens][vocab] fp16, bf16 or fp32 (the same), row strides in elements; the aligned 16 bytes in
 *                          which a row begins and ends are read whole
 *   tokens, parents      : int32 [tokens]; a token outside the vocabulary is rejected
 *   uniforms             : fp32 [tokens] in [0, 1): a node's own number, node 0's draws the new token
 *   temperature          : of all rows, finite and at least 0, or where it is not NULL temperatures fp32 [rows], any: 0 or
 *                          less and NaN are greedy, infinity makes all tokens of finite logits alike
 *   accepted             : int32 [rows], accepted nodes, node 0 among them; 0 without nodes
 *   path, out_tokens     : int32 [rows][max_new]: the accepted nodes; the accepted nodes' tokens after the first's and the
 *                          new token, as many; then -1.  A row of logits with NaN, +inf, or nothing but -inf ends
 *                          the path with -1 as its new token: the sequence has failed, and -1 is no token to go on with.
 * max_new <= BSG_TREE_NODES, vocab <= 2^20, rows <= 16384.  Workspace as bsg_kv_attention.  It has no slots: in a batch some of
 * whose sequences take no part, bsg_verify_drafts_slots (bsgdraft_slots.h) leaves those out. */
int64_t bsg_verify_drafts_workspace_bytes(int64_t tokens, int32_t rows, int64_t vocab, int32_t max_new, int dtype,
                                          int32_t drafts);
int bsg_verify_drafts(const void* logits, int64_t logits_stride, const void* draft_logits, int64_t draft_stride,
                      int64_t tokens, int64_t vocab, const int32_t* token_ids, const float* uniforms,
                      const int32_t* parents, const int32_t* cu, int32_t rows, int32_t max_new, float temperature,
                      const float* temperatures, int32_t* accepted, int32_t* path, int32_t* out_tokens, int dtype, void* ws,
                      int64_t ws_bytes, void* stream);

/* What was accepted of a tree stays in the cache, in every layer of the pool: of the newest n tokens of
 * slot slots[b] (NULL: slot b), n = cu[b+1] - cu[b] (max_new where cu is NULL), those at the places path[b][0 ..
 * accepted[b]) move, in order, to the place of the first; the length shrinks to hold them, the pages past it are released.
 * Of a path only what ascends, from 0 .. n-1, counts.  A token that changes its page is rounded again under that page's
 * scale, which grows as bsg_kv_append's does, the page's other tokens with it; within a page, bytes move.  A page's scale
 * never shrinks: where a rejected token had raised it, the page's other tokens were rounded again under it when that one was
 * appended, the smallest to steps of 2^-9 of the larger scale, and stay so.
 *   pool   : page_bytes = 2 n_heads page_size head_dim and page_scales = 2 n_heads, as bsg_kv_cache
 *   path   : int32 [rows][max_new]
 * Slots must be distinct and the pages of the new tokens a sequence's own; a slot out of range, or of fewer than n
 * tokens, is left as it is.  max_new <= BSG_TREE_NODES, rows <= BSG_PAGES_MAX_ROWS.  Workspace:
 * bsg_pages_keep_workspace_bytes(rows), no initialisation; as in bsg_pages_extend the first of two launches leaves the second
 * its plan there, so threads that share a stream need one each. */
int64_t bsg_pages_keep_workspace_bytes(int32_t rows);
int bsg_pages_keep(const bsg_page_pool* pool, int32_t n_heads, int32_t head_dim, const int32_t* path,
                   const int32_t* accepted, const int32_t* cu, const int32_t* slots, int32_t rows, int32_t max_new,
                   void* ws, int64_t ws_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* BSGDRAFT_H */
