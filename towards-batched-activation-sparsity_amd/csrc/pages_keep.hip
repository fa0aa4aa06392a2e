// pages_keep.hip — what was accepted of a tree of drafted tokens stays in the 8-bit paged cache, beside each other behind the
// tokens before the tree; the rest leaves it (include/bsgdraft.h).
//
// A first launch, a wave a sequence, looks at paths and tables: which tokens move from which place of which page to which,
// and what of the table, lengths and counts changes.  In the second a wave has a head of a layer, which starts from that
// plan, so that scales and bytes come at once.  A token never moves to a place behind its own, nor to one that a later
// token of the path has to be read from, so 64 lanes read as many tokens as they hold, then write them.  A page that
// takes over tokens of a larger scale gets the scale that they need, and what it holds is rounded again, among it the
// tokens that move within it.

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
  int4* plan;                   // [rows][1 + BSG_TREE_NODES]: {moves}, then {source page, target page, place there, place here} in order
  int64_t table_stride, units;  // units of a sequence: layers x heads
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

__global__ __launch_bounds__(64) void bsg_pages_keep_plan_kernel(KeepParams p) {
  const int lane = threadIdx.x, row = blockIdx.x;
  int4* const plan = p.plan + (int64_t)row * (1 + BSG_TREE_NODES);
  const Kept k = kept_of(p, row, lane);
  if (k.slot < 0) {
    if (lane == 0) plan[0] = make_int4(0, 0, 0, 0);
    return;
  }
  const int shift = __builtin_ctz((unsigned)p.page_size), in_page = p.page_size - 1;
  int32_t* const table = p.table + (int64_t)k.slot * p.table_stride;
  // lane i: where token i comes from and goes to
  const int src = k.start + k.node, dst = k.start + lane, len = p.lengths[k.slot];
  bool moves = lane < k.count && k.node != lane;
  int sp = -1, dp = -1;
  if (moves) {
    sp = table[src >> shift], dp = table[dst >> shift];
    moves = sp >= 0 && sp < p.num_pages && dp >= 0 && dp < p.num_pages;
  }
  const uint64_t all = __ballot(moves);
  if (moves) plan[1 + __builtin_popcountll(all & ((1ull << lane) - 1))] = make_int4(sp, dp, src & in_page, dst & in_page);
  if (lane == 0) plan[0] = make_int4(__builtin_popcountll(all), 0, 0, 0);
  // the pages past the new end go back (the wave has read what it needs of the table)
  const int from = (k.start + k.count + in_page) >> shift, to = (len + in_page) >> shift;
  for (int j = from + lane; j < to; j += 64) {
    const int32_t page = table[j];
    table[j] = -1;
    if (page >= 0 && page < p.num_pages) atomicSub(p.refs + page, 1);
  }
  if (lane == 0) p.lengths[k.slot] = k.start + k.count;
}

__device__ __forceinline__ float from_lane(float v, int lane) {
  return as_float(__builtin_amdgcn_ds_bpermute(lane << 2, __builtin_bit_cast(int, v)));
}
__device__ __forceinline__ int from_lane(int v, int lane) { return __builtin_amdgcn_ds_bpermute(lane << 2, v); }

__device__ __forceinline__ u32x4 rescale4(u32x4 v, float ratio) {
  return u32x4{rescale(v.x, ratio), rescale(v.y, ratio), rescale(v.z, ratio), rescale(v.w, ratio)};
}
__device__ __forceinline__ float largest4(uint32_t w, float by) {  // of four cached numbers; a NaN is no maximum
  return fmaxf(fmaxf(__builtin_fabsf(__builtin_amdgcn_cvt_f32_fp8((int)w, 0)), __builtin_fabsf(__builtin_amdgcn_cvt_f32_fp8((int)w, 1))),
               fmaxf(__builtin_fabsf(__builtin_amdgcn_cvt_f32_fp8((int)w, 2)), __builtin_fabsf(__builtin_amdgcn_cvt_f32_fp8((int)w, 3)))) * by;
}

// Tokens move as a wave holds them: of the keys a token is D / 16 lanes' 16 bytes, of the values D / 4 lanes' four
// dwords, of which each has one byte of the token.
template <int D, int KV>
struct Movers {
  static constexpr int LANES = KV == 0 ? D / 16 : D / 4, EACH = 64 / LANES;  // lanes of a token, tokens of a load
  // in flight; few paths move more (64 paths below: 16.2 us, with four loads of the values 16.9, with two and eight 17.9)
  static constexpr int LOADS = KV == 0 ? 1 : 2, TOKENS = LOADS * EACH;
  u32x4 v[LOADS];
  // Offset of a lane's 16 bytes of the token at place t of a page.
  static __device__ __forceinline__ int at(int t, int lane) {
    const int i = lane % LANES;
    return (t >> 4) * 16 * D + (KV == 0 ? (i >> 2) * 1024 + (i & 3) * 256 + (t & 15) * 16 : (i >> 4) * 1024 + (t >> 2 & 3) * 256 + (i & 15) * 16);
  }
  // move: lane i's.  Moves m .. end - 1, as many as are held; returns the next.
  template <typename Bytes>
  __device__ __forceinline__ void load(const int4& move, int m, int end, int lane, const Bytes& bytes) {
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
      if (m + k * EACH >= end) break;
      const int i = m + k * EACH + lane / LANES, from = i < end ? i : m;
      const int page = from_lane(move.x, from), t = from_lane(move.z, from);
      v[k] = u32x4{0u, 0u, 0u, 0u};
      if (i < end) v[k] = *(const u32x4*)(bytes(page) + at(t, lane));
    }
  }
  template <typename Bytes>
  __device__ __forceinline__ void store(const int4& move, float ss, float ds, int m, int end, int lane, const Bytes& bytes) {
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
      if (m + k * EACH >= end) break;
      const int i = m + k * EACH + lane / LANES, from = i < end ? i : m;
      const int page = from_lane(move.y, from), t = from_lane(move.w, from), was = from_lane(move.z, from) & 3;
      const float a = from_lane(ss, from), b = from_lane(ds, from);
      if (i >= end) continue;
      uint8_t* const to = bytes(page) + at(t, lane);
      if constexpr (KV == 0) {
        *(u32x4*)to = a == b ? v[k] : rescale4(v[k], a / b);
      } else {
        uint32_t w = (v[k].x >> (8 * was) & 0xffu) | (v[k].y >> (8 * was) & 0xffu) << 8 | (v[k].z >> (8 * was) & 0xffu) << 16 | v[k].w >> (8 * was) << 24;
        if (a != b) w = rescale(w, a / b);
#pragma unroll
        for (int j = 0; j < 4; ++j) to[4 * j + (t & 3)] = (uint8_t)(w >> (8 * j));
      }
    }
  }
  // The largest magnitude among the lane's numbers.
  __device__ __forceinline__ float top(const int4& move, float ss, int m, int end, int lane) const {
    float r = 0.f;
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
      if (m + k * EACH >= end) break;
      const int i = m + k * EACH + lane / LANES, from = i < end ? i : m;
      const int was = from_lane(move.z, from) & 3;
      const float a = from_lane(ss, from);
      if constexpr (KV == 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) r = fmaxf(r, largest4(v[k][j], a));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) r = fmaxf(r, __builtin_fabsf(__builtin_amdgcn_cvt_f32_fp8((int)(v[k][j] >> (8 * was)), 0)) * a);
      }
    }
    return r;
  }
};

// The keys or the values of a head: all moves, the first of which are held.
template <int D, int KV, typename Bytes, typename Scale>
__device__ __forceinline__ void keep(Movers<D, KV>& held, const int4& move, float ss, float ds, int count, int P, int lane, const Bytes& bytes, const Scale& scale_at) {
  constexpr int TOKENS = Movers<D, KV>::TOKENS;
  if (!__any(lane < count && ss > ds)) {  // no page can need a larger scale
    for (int m = 0; m < count; m += TOKENS) {
      if (m > 0) held.load(move, m, count, lane, bytes);
      held.store(move, ss, ds, m, count, lane, bytes);
    }
    return;
  }
  for (int m = 0; m < count;) {
    // the moves to one page
    const int page = __builtin_amdgcn_readlane(move.y, m);
    const uint64_t others = __ballot(lane >= count || move.y != page) & ~((1ull << m) - 1);
    const int end = others ? __builtin_ctzll(others) : 64;
    const float old = as_float(__builtin_amdgcn_readlane(__builtin_bit_cast(int, ds), m));
    if (__any(lane >= m && lane < end && ss > ds)) {
      float top = 0.f;
      for (int i = m; i < end; i += TOKENS) {
        held.load(move, i, end, lane, bytes);
        top = fmaxf(top, held.top(move, ss, i, end, lane));
      }
      top = fmaxf(top, lane_xor<1>(top)), top = fmaxf(top, lane_xor<2>(top)), top = fmaxf(top, lane_xor<4>(top));
      top = fmaxf(top, lane_xor<8>(top)), top = fmaxf(top, lane_xor<16>(top)), top = fmaxf(top, lane_xor<32>(top));
      const float need = scale_for(top);
      if (need > old) {
        uint8_t* const to = bytes(page);
        const float ratio = old / need;
        for (int e = lane * 16; e < P * D; e += 1024) *(u32x4*)(to + e) = rescale4(*(const u32x4*)(to + e), ratio);
        if (lane == 0) *scale_at(page) = need;
        if (move.x == page) ss = need;
        if (move.y == page) ds = need;
        __builtin_amdgcn_s_waitcnt(0);  // what moves within the page is read from what has just been written
      }
    }
    for (; m < end; m += TOKENS) {
      held.load(move, m, end, lane, bytes);
      held.store(move, ss, ds, m, end, lane, bytes);
    }
    m = end;
  }
}

constexpr int kWaves = 4;

// Latency and half-used sectors bound it: a token's keys are 16 bytes here and there, its values a byte of each dword, so that
// 64 paths in trees of 16, 8 layers x 32 heads, 14 MB, read 33 and write 16: 16 us, after 4 of the plan.  (A work-group a
// sequence and layer, which works out the plan by itself and takes the page through LDS: 28 + 5.)
template <int D>
__global__ __launch_bounds__(64 * kWaves) void bsg_pages_keep_kernel(KeepParams p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t unit = (int64_t)blockIdx.x * kWaves + wave;
  if (unit >= p.units) return;
  const int4* const plan = p.plan + (int64_t)blockIdx.y * (1 + BSG_TREE_NODES);
  int4 move = plan[1 + lane];  // on its way beside the count; what lies past that is nothing yet
  const int count = __builtin_amdgcn_readfirstlane(plan[0].x);
  if (count == 0) return;
  if (lane >= count) move = make_int4(0, 0, 0, 0);
  const int P = p.page_size;
  const int64_t layer = unit / p.heads, head = unit - layer * p.heads;
  const auto index_of = [&](int page) { return ((layer * p.num_pages + page) * p.heads + head) * 2; };
  const auto keys = [&](int page) { return p.pages + index_of(page) * ((int64_t)P * D); };
  const auto values = [&](int page) { return p.pages + (index_of(page) + 1) * ((int64_t)P * D); };
  const f32x2 ss = *(const f32x2*)(p.scales + index_of(move.x)), ds = *(const f32x2*)(p.scales + index_of(move.y));
  Movers<D, 0> k;
  Movers<D, 1> v;
  k.load(move, 0, count, lane, keys);
  v.load(move, 0, count, lane, values);
  keep<D, 0>(k, move, ss.x, ds.x, count, P, lane, keys, [&](int page) { return p.scales + index_of(page); });
  keep<D, 1>(v, move, ss.y, ds.y, count, P, lane, values, [&](int page) { return p.scales + index_of(page) + 1; });
}

}  // namespace

extern "C" int64_t bsg_pages_keep_workspace_bytes(int32_t rows) {
  if (rows < 0 || rows > BSG_PAGES_MAX_ROWS) return -1;
  return (int64_t)rows * (1 + BSG_TREE_NODES) * (int64_t)sizeof(int4);
}

extern "C" int bsg_pages_keep(const bsg_page_pool* pool, int32_t n_heads, int32_t head_dim, const int32_t* path,
                              const int32_t* accepted, const int32_t* cu, const int32_t* slots, int32_t rows,
                              int32_t max_new, void* ws, int64_t ws_bytes, void* stream) {
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
  const int64_t need = bsg_pages_keep_workspace_bytes(rows);
  if (!ws || ws_bytes < need)
    return fail(BSG_ERR_WORKSPACE, "workspace of %lld bytes, %lld needed", (long long)ws_bytes, (long long)need);
  if (!is_aligned(ws, 16)) return fail(BSG_ERR_ALIGN, "workspace must be 16-byte aligned");
  KeepParams p;
  p.plan = (int4*)ws;
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
  p.units = pool->layers * n_heads;
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
  hipLaunchKernelGGL(bsg_pages_keep_plan_kernel, dim3((unsigned)rows), dim3(64), 0, st, p);
  if (head_dim == 64) hipLaunchKernelGGL((bsg_pages_keep_kernel<64>), grid, dim3(64 * kWaves), 0, st, p);
  else hipLaunchKernelGGL((bsg_pages_keep_kernel<128>), grid, dim3(64 * kWaves), 0, st, p);
  return launch_status("bsg_pages_keep");
}
