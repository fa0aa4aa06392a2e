// kv_attention.hip — attention of each sequence's newest tokens over its cached ones (include/bsgserve.h): the
// entry points, and how a call is cut.  The kernels are kv_attention.hpp's.

#include "kv_attention.hpp"

namespace {

constexpr int kPrefillRows = 32;  // a cached head's rows past which the prefill kernel runs

// How a call is cut.  Few work-groups leave most compute units idle unless the long axis is split, to
// two for each unit and at least 256 tokens a part.  A part of 128 rows writes and reads 66 KiB, so
// there only where units would have none at all, and not over less than 1024 tokens (a prompt of 500
// alone: 21.0 us, 23.8 in two parts; 2 x 40 tokens over 1500: 22.4 us in six, 31.5 in two).
Shape shape_of(int32_t rows, int32_t kv_heads, int32_t group, int32_t max_new, int64_t max_len, int32_t cus) {
  Shape s;
  const int64_t per_head = (int64_t)max_new * group;
  s.rows = per_head <= 16 ? 16 : per_head <= kPrefillRows ? 32 : 128;
  s.row_tiles = (int32_t)ceil_div(per_head, s.rows);
  const int64_t tiles = (int64_t)rows * kv_heads * s.row_tiles;
  if (max_len < 1) max_len = 1;
  int64_t want = ceil_div((int64_t)2 * cus, tiles > 0 ? tiles : 1);
  if (want > kMaxSplits) want = kMaxSplits;
  if (want > ceil_div(max_len, 256)) want = ceil_div(max_len, 256);
  if (s.rows == 128 && (tiles >= cus || max_len < 1024)) want = 1;
  if (tiles * 4 > BSG_KV_COUNTER_BYTES) want = 1;
  s.chunk = (int32_t)(ceil_div(ceil_div(max_len, want), 128) * 128);
  s.splits = (int32_t)ceil_div(max_len, s.chunk);
  return s;
}

template <typename T, int D>
void launch(const AttnParams& p, const Shape& s, dim3 grid, hipStream_t st) {
  switch (s.rows) {
    case 16: hipLaunchKernelGGL((bsg_kv_attention_kernel<T, D, 1, false>), grid, dim3(256), 0, st, p); break;
    case 32: hipLaunchKernelGGL((bsg_kv_attention_kernel<T, D, 2, false>), grid, dim3(256), 0, st, p); break;
    default: hipLaunchKernelGGL((bsg_kv_prefill_kernel<T, D, false>), grid, dim3(256), 0, st, p); break;
  }
}

}  // namespace

extern "C" int64_t bsg_kv_attention_workspace_bytes(const bsg_kv_cache* cache, int32_t rows, int32_t q_heads,
                                                    int32_t max_new, int64_t max_len, int32_t cu_count) {
  if (check_kv_cache(cache) || check_heads(cache, q_heads) || rows < 0 || max_new < 0 || cu_count < 1) return -1;
  const int64_t most = (int64_t)cache->max_pages * cache->page_size;
  if (max_len <= 0 || max_len > most) max_len = most;
  return workspace_bytes(shape_of(rows, cache->n_heads, q_heads / cache->n_heads, max_new, max_len, cu_count), rows,
                         cache->n_heads, cache->head_dim);
}

extern "C" int bsg_kv_attention(const void* q, int64_t q_stride_t, int64_t q_stride_h, int64_t tokens,
                                int32_t q_heads, const bsg_kv_cache* cache, const int32_t* slots, int32_t rows,
                                const int32_t* cu, int32_t max_new, int64_t max_len, float sm_scale, void* out,
                                int64_t o_stride_t, int64_t o_stride_h, float* lse, int dtype, void* ws,
                                int64_t ws_bytes, int32_t cu_count, void* stream) {
  const AttnCall c = {q, q_stride_t, q_stride_h, tokens, q_heads, cache, slots, rows, cu, max_new, sm_scale, out,
                      o_stride_t, o_stride_h, lse, dtype, ws, ws_bytes, cu_count};
  if (const int rc = check_call(c)) return rc;
  if (tokens == 0 || rows == 0 || max_new == 0) return BSG_OK;
  if (const int rc = check_tensors(c)) return rc;
  const int64_t most = (int64_t)cache->max_pages * cache->page_size;
  if (max_len <= 0 || max_len > most) max_len = most;
  const Shape s = shape_of(rows, cache->n_heads, q_heads / cache->n_heads, max_new, max_len, cu_count);
  AttnParams p;
  if (const int rc = call_params(c, s, &p)) return rc;
  const dim3 grid((unsigned)(cache->n_heads * s.row_tiles), (unsigned)s.splits, (unsigned)rows);
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == BSG_F16)
    cache->head_dim == 64 ? launch<_Float16, 64>(p, s, grid, st) : launch<_Float16, 128>(p, s, grid, st);
  else
    cache->head_dim == 64 ? launch<__bf16, 64>(p, s, grid, st) : launch<__bf16, 128>(p, s, grid, st);
  return launch_status("bsg_kv_attention");
}
