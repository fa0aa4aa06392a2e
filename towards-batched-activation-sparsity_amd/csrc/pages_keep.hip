// pages_keep.hip — what was accepted of a tree of drafted tokens stays in the 8-bit paged cache, beside each other behind the
// tokens before the tree; the rest leaves it (include/bsgdraft.h).
//
// A wave has the keys or the values of one head, layer and sequence.  It reads all that moves into LDS before it
// writes, since one token's new place can be another's old one; a page that takes over tokens from another one of a
// larger scale gets the scale that they need, and what it holds is rounded again.  A second launch shortens the tables,
// which the first one reads.

#include "bsgdraft.h"
#include "kv_quant.hpp"

using namespace bsgk;

namespace bsgk {
int check_kv_cache(const bsg_kv_cache* c);
}

namespace {

struct KeepParams {
  uint8_t* pages;
  float* scales;
  int32_t* table;
  int32_t* lengths;
  int32_t* refs;
  const int32_t* path;
  const int32_t* accepted;
  const int32_t* cu;
  const int32_t* slots;
  int64_t table_stride, units;  // units of a sequence: layers x heads x 2
  int32_t num_pages, page_size, num_slots, max_pages, heads, rows, max_new;
};

// A sequence's drafts: where they begin, and how many of its path count.  Lane i of a wave has path[i].
struct Kept {
  int slot, start, count;
  int node;  // the place, among the drafts, of the token that goes to place `lane`
};
__device__ __forceinline__ Kept kept_of(const KeepParams& p, int row, int lane) {
  Kept k;
  k.slot = p.slots ? p.slots[row] : row;
  const int want = p.accepted[row];
  k.node = lane < p.max_new ? p.path[(int64_t)row * p.max_new + lane] : -1;
  int n = p.max_new;
  if (p.cu) n = p.cu[row + 1] - p.cu[row];
  int len = -1;
  if (k.slot >= 0 && k.slot < p.num_slots) len = p.lengths[k.slot];
  const int64_t most = (int64_t)p.max_pages * p.page_size;
  k.start = len - n, k.count = 0;
  if (n < 0 || k.start < 0 || len > most) {
    k.slot = -1;
    return k;
  }
  const int before = __shfl_up(k.node, 1);
  const bool good = lane < want && lane < p.max_new && k.node >= 0 && k.node < n && (lane == 0 || k.node > before);
  const uint64_t bad = ~__ballot(good);
  k.count = bad == 0 ? 64 : __builtin_ctzll(bad);
  return k;
}

constexpr int kWaves = 4;

template <int D>
__global__ __launch_bounds__(64 * kWaves) void bsg_pages_keep_kernel(KeepParams p) {
  constexpr int C = D / 64;
  __shared__ uint8_t s_bytes[kWaves][BSG_TREE_NODES][D];  // the tokens on their way
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = blockIdx.y;
  const int64_t unit = (int64_t)blockIdx.x * kWaves + wave;
  if (unit >= p.units) return;
  const Kept k = kept_of(p, row, lane);
  if (k.slot < 0) return;
  // lane i: where token i comes from and goes to
  bool moves = lane < k.count && k.node != lane;
  if (!__any(moves)) return;
  const int P = p.page_size, shift = __builtin_ctz((unsigned)P);
  const int kv = (int)(unit & 1);
  const int64_t block = unit >> 1, layer = block / p.heads, head = block - layer * p.heads;
  const int src = k.start + k.node, dst = k.start + lane;
  int sp = -1, dp = -1;
  if (moves) {
    const int32_t* const at = p.table + (int64_t)k.slot * p.table_stride;
    sp = at[src >> shift], dp = at[dst >> shift];
    moves = sp >= 0 && sp < p.num_pages && dp >= 0 && dp < p.num_pages;
  }
  const auto index_of = [&](int page) { return ((layer * p.num_pages + page) * p.heads + head) * 2 + kv; };
  float ss = 1.f, ds = 1.f;
  if (moves) ss = p.scales[index_of(sp)], ds = p.scales[index_of(dp)];
  // byte of channel x of the token at place t of a page
  const auto place = [&](int t, int x) {
    const int r = x & 63;
    return (t >> 4) * 16 * D + (x >> 6) * 1024 +
           (kv == 0 ? (r >> 4) * 256 + (t & 15) * 16 + (r & 15) : (t >> 2 & 3) * 256 + (r & 15) * 16 + (r >> 4) * 4 + (t & 3));
  };
  uint64_t left = __ballot(moves);
  for (uint64_t m = left; m; m &= m - 1) {
    const int i = __builtin_ctzll(m);
    const uint8_t* const at = p.pages + index_of(__builtin_amdgcn_readlane(sp, i)) * ((int64_t)P * D);
    const int t = __builtin_amdgcn_readlane(src, i) & (P - 1);
#pragma unroll
    for (int c = 0; c < C; ++c) s_bytes[wave][i][64 * c + lane] = at[place(t, 64 * c + lane)];
  }
  while (left) {
    // the tokens that go to one page; the lane that wrote a byte reads it
    const int first = __builtin_ctzll(left);
    const int page = __builtin_amdgcn_readlane(dp, first);
    const uint64_t mine = left & __ballot(moves && dp == page);
    left &= ~mine;
    float top = 0.f;
    for (uint64_t m = mine; m; m &= m - 1) {
      const int i = __builtin_ctzll(m);
      const float by = as_float(__builtin_amdgcn_readlane(__builtin_bit_cast(int, ss), i));
#pragma unroll
      for (int c = 0; c < C; ++c)
        top = fmaxf(top, __builtin_fabsf(__builtin_amdgcn_cvt_f32_fp8((int)s_bytes[wave][i][64 * c + lane], 0)) * by);  // a NaN is no maximum
    }
    for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
    const float old = as_float(__builtin_amdgcn_readlane(__builtin_bit_cast(int, ds), first));
    const float need = scale_for(top), scale = need > old ? need : old;
    uint8_t* const to = p.pages + index_of(page) * ((int64_t)P * D);
    if (scale != old) {
      const float ratio = old / scale;
      for (int e = lane * 16; e < P * D; e += 1024) {
        u32x4* const at = (u32x4*)(to + e);
        const u32x4 v = *at;
        *at = u32x4{rescale(v.x, ratio), rescale(v.y, ratio), rescale(v.z, ratio), rescale(v.w, ratio)};
      }
      if (lane == 0) p.scales[index_of(page)] = scale;
      __builtin_amdgcn_s_waitcnt(0);  // the tokens go into what has just been written
    }
    for (uint64_t m = mine; m; m &= m - 1) {
      const int i = __builtin_ctzll(m);
      const int t = __builtin_amdgcn_readlane(dst, i) & (P - 1);
      const float was = as_float(__builtin_amdgcn_readlane(__builtin_bit_cast(int, ss), i));
#pragma unroll
      for (int c = 0; c < C; ++c) {
        uint32_t b = s_bytes[wave][i][64 * c + lane];
        if (was != scale) b = rescale(b, was / scale);
        to[place(t, 64 * c + lane)] = (uint8_t)b;
      }
    }
  }
}

// A wave a sequence: its length, its table row from the first page that holds nothing any more, those pages' counts.
__global__ __launch_bounds__(64) void bsg_pages_keep_table_kernel(KeepParams p) {
  const int lane = threadIdx.x, row = blockIdx.x;
  const Kept k = kept_of(p, row, lane);
  if (k.slot < 0) return;
  const int len = p.lengths[k.slot], shift = __builtin_ctz((unsigned)p.page_size);
  const int from = (k.start + k.count + p.page_size - 1) >> shift, to = (len + p.page_size - 1) >> shift;
  int32_t* const at = p.table + (int64_t)k.slot * p.table_stride;
  for (int j = from + lane; j < to; j += 64) {
    const int32_t page = at[j];
    at[j] = -1;
    if (page >= 0 && page < p.num_pages) atomicSub(p.refs + page, 1);
  }
  if (lane == 0) p.lengths[k.slot] = k.start + k.count;
}

}  // namespace

extern "C" int bsg_pages_keep(const bsg_page_pool* pool, int32_t n_heads, int32_t head_dim, const int32_t* path,
                              const int32_t* accepted, const int32_t* cu, const int32_t* slots, int32_t rows,
                              int32_t max_new, void* stream) {
  if (!pool) return fail(BSG_ERR_ARG, "pool is null");
  if (!pool->pages || !pool->scales || !pool->page_table || !pool->lengths || !pool->refcounts)
    return fail(BSG_ERR_ARG, "pool: null pointer (pages=%p scales=%p page_table=%p lengths=%p refcounts=%p)", pool->pages,
                (void*)pool->scales, (void*)pool->page_table, (void*)pool->lengths, (void*)pool->refcounts);
  // the sizes of what a layer of the pool is as a cache
  const bsg_kv_cache cache = {pool->pages, pool->scales, pool->num_pages, n_heads, pool->page_size, head_dim, pool->num_slots,
                              pool->max_pages, pool->table_stride, pool->page_table, pool->lengths};
  if (const int rc = check_kv_cache(&cache)) return rc;
  if (pool->layers < 1 || pool->page_bytes != (int64_t)2 * n_heads * pool->page_size * head_dim || pool->page_scales != 2 * (int64_t)n_heads)
    return fail(BSG_ERR_ARG, "pool: layers=%lld page_bytes=%lld page_scales=%lld with %d heads of %d", (long long)pool->layers,
                (long long)pool->page_bytes, (long long)pool->page_scales, n_heads, head_dim);
  if (rows < 0 || max_new < 0) return fail(BSG_ERR_ARG, "rows=%d max_new=%d", rows, max_new);
  if (rows > BSG_PAGES_MAX_ROWS) return fail(BSG_ERR_UNSUPPORTED, "%d slots in one call (at most %d)", rows, BSG_PAGES_MAX_ROWS);
  if (max_new > BSG_TREE_NODES) return fail(BSG_ERR_UNSUPPORTED, "%d nodes in a tree (at most %d)", max_new, BSG_TREE_NODES);
  if (!slots && rows > pool->num_slots) return fail(BSG_ERR_ARG, "%d rows, %d slots", rows, pool->num_slots);
  if (rows == 0) return BSG_OK;
  if (!accepted || (!path && max_new > 0))
    return fail(BSG_ERR_ARG, "null pointer (path=%p accepted=%p)", (const void*)path, (const void*)accepted);
  KeepParams p;
  p.pages = (uint8_t*)pool->pages;
  p.scales = pool->scales;
  p.table = pool->page_table;
  p.lengths = pool->lengths;
  p.refs = pool->refcounts;
  p.path = path;
  p.accepted = accepted;
  p.cu = cu;
  p.slots = slots;
  p.table_stride = pool->table_stride;
  p.units = pool->layers * n_heads * 2;
  p.num_pages = (int32_t)pool->num_pages;
  p.page_size = pool->page_size;
  p.num_slots = pool->num_slots;
  p.max_pages = pool->max_pages;
  p.heads = n_heads;
  p.rows = rows;
  p.max_new = max_new;
  const int64_t gx = ceil_div(p.units, kWaves);
  if (gx > kLaunchGroups / BSG_PAGES_MAX_ROWS) return fail(BSG_ERR_UNSUPPORTED, "pool: %lld layers of %d heads", (long long)pool->layers, n_heads);
  const hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)gx, (unsigned)rows);
  if (head_dim == 64) hipLaunchKernelGGL((bsg_pages_keep_kernel<64>), grid, dim3(64 * kWaves), 0, st, p);
  else hipLaunchKernelGGL((bsg_pages_keep_kernel<128>), grid, dim3(64 * kWaves), 0, st, p);
  hipLaunchKernelGGL(bsg_pages_keep_table_kernel, dim3((unsigned)rows), dim3(64), 0, st, p);
  return launch_status("bsg_pages_keep");
}
