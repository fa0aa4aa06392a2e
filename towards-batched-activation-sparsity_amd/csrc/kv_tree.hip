// kv_tree.hip — attention of a tree of drafted tokens over the 8-bit paged cache (include/bsgdraft.h).
//
// The kernels are kv_attention.hpp's with another question of what a row sees: all tokens before the tree, and of
// the tree the row's own node and its ancestors, which each wave works out once, one bit for each of 64 nodes.  Only the
// last steps hold nodes, so only they look at the bits.

#include "bsgdraft.h"
#include "kv_attention.hpp"

namespace {

constexpr int kTileRows = 32;  // a cached head's rows past which tiles of 128 rows run

Shape tree_shape(int32_t rows, int32_t kv_heads, int32_t group, int32_t max_new, int64_t max_len, int32_t cus) {
  Shape s;
  const int64_t per_head = (int64_t)max_new * group;
  s.rows = per_head <= 16 ? 16 : per_head <= kTileRows ? 32 : 128;
  s.row_tiles = (int32_t)ceil_div(per_head, s.rows);
  const int64_t tiles = (int64_t)rows * kv_heads * s.row_tiles;
  if (max_len < 1) max_len = 1;
  int64_t want = ceil_div((int64_t)2 * cus, tiles > 0 ? tiles : 1);
  if (want > kMaxSplits) want = kMaxSplits;
  if (want > ceil_div(max_len, 256)) want = ceil_div(max_len, 256);
  if (tiles * 4 > BSG_KV_COUNTER_BYTES) want = 1;
  s.chunk = (int32_t)(ceil_div(ceil_div(max_len, want), 128) * 128);
  s.splits = (int32_t)ceil_div(max_len, s.chunk);
  return s;
}

template <typename T, int D>
void launch(const AttnParams& p, const Shape& s, dim3 grid, hipStream_t st) {
  switch (s.rows) {
    case 16: hipLaunchKernelGGL((bsg_kv_attention_kernel<T, D, 1, true>), grid, dim3(256), 0, st, p); break;
    case 32: hipLaunchKernelGGL((bsg_kv_attention_kernel<T, D, 2, true>), grid, dim3(256), 0, st, p); break;
    default: hipLaunchKernelGGL((bsg_kv_prefill_kernel<T, D, true>), grid, dim3(256), 0, st, p); break;
  }
}

int check_nodes(int32_t max_new) {
  if (max_new > BSG_TREE_NODES) return fail(BSG_ERR_UNSUPPORTED, "%d nodes in a tree (at most %d)", max_new, BSG_TREE_NODES);
  return BSG_OK;
}

}  // namespace

extern "C" int64_t bsg_kv_tree_attention_workspace_bytes(const bsg_kv_cache* cache, int32_t rows, int32_t q_heads,
                                                         int32_t max_new, int64_t max_len, int32_t cu_count) {
  if (check_kv_cache(cache) || check_heads(cache, q_heads) || rows < 0 || max_new < 0 || check_nodes(max_new) || cu_count < 1)
    return -1;
  const int64_t most = (int64_t)cache->max_pages * cache->page_size;
  if (max_len <= 0 || max_len > most) max_len = most;
  return workspace_bytes(tree_shape(rows, cache->n_heads, q_heads / cache->n_heads, max_new, max_len, cu_count), rows,
                         cache->n_heads, cache->head_dim);
}

extern "C" int bsg_kv_tree_attention(const void* q, int64_t q_stride_t, int64_t q_stride_h, int64_t tokens,
                                     int32_t q_heads, const int32_t* parents, const bsg_kv_cache* cache,
                                     const int32_t* slots, int32_t rows, const int32_t* cu, int32_t max_new,
                                     int64_t max_len, float sm_scale, void* out, int64_t o_stride_t, int64_t o_stride_h,
                                     float* lse, int dtype, void* ws, int64_t ws_bytes, int32_t cu_count, void* stream) {
  const AttnCall c = {q, q_stride_t, q_stride_h, tokens, q_heads, cache, slots, rows, cu, max_new, sm_scale, out,
                      o_stride_t, o_stride_h, lse, dtype, ws, ws_bytes, cu_count};
  if (const int rc = check_call(c)) return rc;
  if (const int rc = check_nodes(max_new)) return rc;
  if (tokens == 0 || rows == 0 || max_new == 0) return BSG_OK;
  if (!parents) return fail(BSG_ERR_ARG, "parents is null");
  if (const int rc = check_tensors(c)) return rc;
  const int64_t most = (int64_t)cache->max_pages * cache->page_size;
  if (max_len <= 0 || max_len > most) max_len = most;
  const Shape s = tree_shape(rows, cache->n_heads, q_heads / cache->n_heads, max_new, max_len, cu_count);
  AttnParams p;
  if (const int rc = call_params(c, s, &p)) return rc;
  p.parents = parents;
  const dim3 grid((unsigned)(cache->n_heads * s.row_tiles), (unsigned)s.splits, (unsigned)rows);
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == BSG_F16)
    cache->head_dim == 64 ? launch<_Float16, 64>(p, s, grid, st) : launch<_Float16, 128>(p, s, grid, st);
  else
    cache->head_dim == 64 ? launch<__bf16, 64>(p, s, grid, st) : launch<__bf16, 128>(p, s, grid, st);
  return launch_status("bsg_kv_tree_attention");
}
