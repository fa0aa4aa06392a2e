// pages.hip — the pages of a paged cache (include/bsgserve.h): copying, forking, extending, freeing
// and compacting them on the device.
//
// Page ids, counts and tables never come to the host.  What decides over pages in order (which are
// free, which row gets which) is one work-group's scan over the counts; what moves data is a second
// launch that takes the pairs from the workspace and copies at the rate of HBM.  All results are
// whole numbers and do not depend on the order in which work-groups run.

#include "serve.hpp"

using namespace bsgk;

namespace {

struct Pool {
  uint8_t* pages;
  float* scales;
  int32_t* table;
  int32_t* lengths;
  int32_t* refs;
  int64_t layers, page_bytes, page_scales, table_stride;
  int32_t num_pages, page_size, num_slots, max_pages;
};

__device__ __forceinline__ bool is_page(const Pool& p, int32_t id) { return id >= 0 && id < p.num_pages; }
__device__ __forceinline__ bool is_slot(const Pool& p, int32_t s) { return s >= 0 && s < p.num_slots; }

// Pages move in pieces of 16 KiB, one for each work-group of 256 threads: four 16-byte loads in flight
// for each thread, and enough work-groups for the machine from a few pages on.  Against one
// work-group a page of 128 KiB: 28 copies x 4 layers 10.9 -> 9.8 us, 365 MB in and out 73 -> 66
// (5.6 TB/s; a plain copy reaches 5.0).
constexpr int64_t kPiece = 16384;
constexpr int64_t kCopyGroups = 4096;  // of a data-moving launch: every compute unit several times over
__host__ __device__ inline int64_t pieces_of(int64_t page_bytes) { return (page_bytes + kPiece - 1) / kPiece; }

__device__ __forceinline__ void copy_piece(const Pool& p, int64_t layer, int32_t src, int32_t dst, int64_t piece) {
  const int64_t base = layer * p.num_pages;
  const int64_t first = piece * (kPiece / 16) + threadIdx.x, n = p.page_bytes >> 4;
  const u32x4* const from = (const u32x4*)(p.pages + (base + src) * p.page_bytes);
  u32x4* const to = (u32x4*)(p.pages + (base + dst) * p.page_bytes);
  u32x4 v[4];
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (first + 256 * k < n) v[k] = __builtin_nontemporal_load(from + first + 256 * k);
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (first + 256 * k < n) __builtin_nontemporal_store(v[k], to + first + 256 * k);
  if (piece == 0) {
    const float* const sf = p.scales + (base + src) * p.page_scales;
    float* const st = p.scales + (base + dst) * p.page_scales;
    for (int64_t i = threadIdx.x; i < p.page_scales; i += 256) st[i] = sf[i];
  }
}

__global__ __launch_bounds__(256) void bsg_pages_copy_kernel(Pool p, const int32_t* __restrict__ src,
                                                             const int32_t* __restrict__ dst, int32_t n) {
  const int64_t pieces = pieces_of(p.page_bytes), each = p.layers * pieces;
  for (int64_t item = blockIdx.x; item < n * each; item += gridDim.x) {
    const int64_t i = item / each, part = item - i * each, layer = part / pieces;
    const int32_t s = src[i], d = dst[i];
    if (is_page(p, s) && is_page(p, d) && s != d) copy_piece(p, layer, s, d, part - layer * pieces);
  }
}

// ---------------------------------------------------------------------------------------------- fork

constexpr int kForkCols = 8;  // table columns of one work-group: 1024 pairs x 8 x 4 bytes of LDS

// 64 pairs over 20 columns: 7.7 us, a chain of pairs, entries, counts.  Every entry that a work-group overwrites lies in its own columns, and it has read them all, the
// parents' and the children's, before a barrier, after which it writes.
__global__ __launch_bounds__(256) void bsg_pages_fork_kernel(Pool p, const int32_t* __restrict__ parents,
                                                             const int32_t* __restrict__ children, int32_t n) {
  constexpr int PER = BSG_PAGES_MAX_ROWS / 256;
  __shared__ alignas(16) int32_t s_child[BSG_PAGES_MAX_ROWS + 4];
  __shared__ int32_t s_parent[BSG_PAGES_MAX_ROWS];
  __shared__ int32_t s_new[BSG_PAGES_MAX_ROWS * kForkCols], s_old[BSG_PAGES_MAX_ROWS * kForkCols];
  const int tid = threadIdx.x;
  const int c0 = blockIdx.x * kForkCols;
  for (int i = tid; i < ((n + 3) & ~3); i += 256) {
    const int32_t c = i < n ? children[i] : -1, a = i < n ? parents[i] : -1;
    s_child[i] = is_slot(p, c) && is_slot(p, a) ? c : -1;
    s_parent[i] = a;
  }
  __syncthreads();
  const bool lengths = c0 >= p.max_pages;  // the work-group past the columns moves the lengths
  const int cols = lengths ? 1 : p.max_pages - c0 < kForkCols ? p.max_pages - c0 : kForkCols;
  for (int e = tid; e < n * cols; e += 256) {
    const int i = e / cols, c = e - i * cols;
    if (s_child[i] >= 0) {
      s_new[e] = lengths ? p.lengths[s_parent[i]] : p.table[s_parent[i] * p.table_stride + c0 + c];
      s_old[e] = lengths ? p.lengths[s_child[i]] : p.table[s_child[i] * p.table_stride + c0 + c];
    }
  }
  // of pairs with the same child the last one counts
  bool lost[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int i = tid + 256 * k;
    lost[k] = false;
    if (i < n && s_child[i] >= 0) {
      const int32_t c = s_child[i];
      for (int j = i & ~3; j < n; j += 4) {
        const int4 v = *(const int4*)(s_child + j);
        lost[k] |= (v.x == c && j > i) || (v.y == c && j + 1 > i) || (v.z == c && j + 2 > i) || (v.w == c && j + 3 > i);
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < PER; ++k)
    if (lost[k]) s_child[tid + 256 * k] = -1;
  __syncthreads();
  for (int e = tid; e < n * cols; e += 256) {
    const int i = e / cols, c = e - i * cols;
    if (s_child[i] < 0) continue;
    int32_t* const at = lengths ? p.lengths + s_child[i] : p.table + s_child[i] * p.table_stride + c0 + c;
    const int32_t was = s_old[e], now = s_new[e];
    if (was == now) continue;
    *at = now;
    if (lengths) continue;
    if (is_page(p, was)) atomicSub(p.refs + was, 1);
    if (is_page(p, now)) atomicAdd(p.refs + now, 1);
  }
}

// ---------------------------------------------------------------------------------------------- free

// An entry is taken out by an exchange, so that a slot named twice releases its pages once.  24 slots of
// 44 pages: 3.0 us.
__global__ __launch_bounds__(256) void bsg_pages_free_kernel(Pool p, const int32_t* __restrict__ slots) {
  const int32_t slot = slots[blockIdx.x];
  if (!is_slot(p, slot)) return;
  const int c = blockIdx.y * 256 + threadIdx.x;
  if (c < p.max_pages) {
    const int32_t was = atomicExch(p.table + slot * p.table_stride + c, -1);
    if (is_page(p, was)) atomicSub(p.refs + was, 1);
  }
  if (c == 0) p.lengths[slot] = 0;
}

// ---------------------------------------------------------------------------------------------- scans

constexpr int kScan = 1024;  // threads of a scanning work-group

// Sum of `v` over the threads before this one; *total gets the sum over all (kScan threads).
__device__ __forceinline__ int block_scan(int v, int* total) {
  __shared__ int s_wave[kScan / 64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int y = __shfl_up(x, m);
    if (lane >= m) x += y;
  }
  __syncthreads();
  if (lane == 63) s_wave[w] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kScan / 64; ++i) {
    const int t = s_wave[i];
    before += i < w ? t : 0;
    all += t;
  }
  *total = all;
  return before + x - v;
}

// The counts of 4 pages per thread, kept in groups of consecutive ids.
__device__ __forceinline__ void load_counts(const Pool& p, int64_t id, int32_t v[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = id + k < p.num_pages ? p.refs[id + k] : -1;  // -1: no such page
}

// Workspace of a plan: a header, then lists of num_pages entries.
struct Row {  // what bsg_pages_extend decided for a row
  int32_t slot, have, fresh, first, copy_from, length, pad0, pad1;
};
constexpr int64_t kHeader = 256, kRows = BSG_PAGES_MAX_ROWS * sizeof(Row);

// ---------------------------------------------------------------------------------------------- extend

__global__ __launch_bounds__(kScan) void bsg_pages_extend_plan_kernel(Pool p, const int32_t* __restrict__ slots,
                                                                      const int32_t* __restrict__ new_tokens, int32_t n,
                                                                      int32_t* __restrict__ served, Row* __restrict__ rows,
                                                                      int32_t* __restrict__ free_ids) {
  __shared__ int32_t s_tail[kScan];
  const int i = threadIdx.x;
  int32_t v[4];
  load_counts(p, 4 * i, v);  // the first free pages are mostly here: on their way while the rows are weighed
  const int32_t slot = i < n ? (slots ? slots[i] : i) : -1;
  const bool real = is_slot(p, slot);
  int64_t len = real ? p.lengths[slot] : 0;
  int64_t add = real ? new_tokens[i] : 0;
  if (add < 0) add = 0;
  if (len < 0) len = 0;
  const int64_t have = (len + p.page_size - 1) / p.page_size, want = (len + add + p.page_size - 1) / p.page_size;
  const bool fits = real && want <= p.max_pages && want - have < 0x1fffff;  // 1024 such sums stay within 32 bits
  const bool inside = fits && add > 0 && len % p.page_size != 0;
  const int32_t tail = inside ? p.table[slot * p.table_stride + have - 1] : -1;
  const int readers = is_page(p, tail) ? p.refs[tail] : 1;
  s_tail[i] = tail;
  __syncthreads();
  int earlier = 0;
  if (readers > 1)
    for (int j = 0; j < i; ++j) earlier += s_tail[j] == tail;
  const bool split = readers - earlier > 1;
  const int need = fits ? (int)(want - have) + split : 0;
  int total;
  const int first = block_scan(need, &total);
  // the free pages, lowest first, until there are enough
  int found = 0;
  for (int64_t base = 0; base < p.num_pages && found < total; base += 4 * kScan) {
    if (base > 0) load_counts(p, base + 4 * i, v);
    const int mine = (v[0] == 0) + (v[1] == 0) + (v[2] == 0) + (v[3] == 0);
    int all;
    int at = found + block_scan(mine, &all);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (v[k] == 0) free_ids[at++] = (int32_t)base + 4 * i + k;
    found += all;
  }
  const bool ok = fits && (first + need <= found || (need == 0 && readers <= 1));
  if (i < n) {
    served[i] = ok;
    rows[i] = Row{ok ? slot : -1, (int32_t)have, ok ? (int32_t)(want - have) : 0, first, ok && split ? tail : -1,
                  (int32_t)(len + add), 0, 0};
  }
}

// Work-group (i, chunk): a part of the copied page's layers; the first chunk also writes row i.  64 rows, some
// 22 pages of 128 KiB copied in 4 layers each (23 MB in and out): 8-10 us after a plan of 5.3, a chain of length,
// entry, count and two scans in one work-group.
__global__ __launch_bounds__(256) void bsg_pages_extend_kernel(Pool p, const Row* __restrict__ rows,
                                                               const int32_t* __restrict__ free_ids) {
  const Row r = rows[blockIdx.x];
  if (r.slot < 0) return;
  const bool split = r.copy_from >= 0;
  const int32_t dst = split ? free_ids[r.first] : -1;
  if (blockIdx.y == 0) {
    int32_t* const row = p.table + r.slot * p.table_stride;
    for (int k = threadIdx.x; k < r.fresh; k += 256) {
      const int32_t id = free_ids[r.first + split + k];
      row[r.have + k] = id;
      p.refs[id] = 1;
    }
    if (threadIdx.x == 0) {
      p.lengths[r.slot] = r.length;
      if (split) {
        row[r.have - 1] = dst;
        p.refs[dst] = 1;
        atomicSub(p.refs + r.copy_from, 1);
      }
    }
  }
  const int64_t pieces = pieces_of(p.page_bytes);
  if (split)
    for (int64_t part = blockIdx.y; part < p.layers * pieces; part += gridDim.y)
      copy_piece(p, part / pieces, r.copy_from, dst, part % pieces);
}

// ---------------------------------------------------------------------------------------------- compact

// In one work-group, 3.3 us for 2000 pages: no more than a few reads of the counts.
// Live and free ids in ascending order; of `live` live pages the moved ones are the last of the
// live list, and they go to the first of the free list.
__global__ __launch_bounds__(kScan) void bsg_pages_compact_plan_kernel(Pool p, int32_t* __restrict__ counts,
                                                                       int32_t* __restrict__ header,
                                                                       int32_t* __restrict__ live_ids,
                                                                       int32_t* __restrict__ free_ids) {
  const int i = threadIdx.x;
  int live = 0;
  for (int64_t base = 0; base < p.num_pages; base += 4 * kScan) {
    int32_t v[4];
    load_counts(p, base + 4 * i, v);
    const int mine = (v[0] > 0) + (v[1] > 0) + (v[2] > 0) + (v[3] > 0);
    int all;
    int at = live + block_scan(mine, &all);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t id = base + 4 * i + k;
      if (v[k] > 0) live_ids[at++] = (int32_t)id;
      else if (id < p.num_pages) free_ids[id - at] = (int32_t)id;
    }
    live += all;
  }
  __syncthreads();  // the lists are written and read by this work-group only
  int moved = 0;
  for (int64_t base = 0; base < p.num_pages - live; base += kScan) {
    int all;
    block_scan(base + i < p.num_pages - live && free_ids[base + i] < live, &all);
    moved += all;
    if (all < kScan) break;
  }
  if (i == 0) {
    counts[0] = live, counts[1] = moved;
    header[0] = live, header[1] = moved;
  }
}

__global__ __launch_bounds__(256) void bsg_pages_compact_kernel(Pool p, const int32_t* __restrict__ header,
                                                                const int32_t* __restrict__ live_ids,
                                                                const int32_t* __restrict__ free_ids) {
  const int32_t live = header[0], moved = header[1];
  const int32_t* const src = live_ids + (live - moved);
  // table entries: the rank of a moved page among the moved ones, by bisection
  const int64_t entries = (int64_t)p.num_slots * p.max_pages;
  if (moved > 0)
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < entries; e += (int64_t)gridDim.x * 256) {
      const int64_t slot = e / p.max_pages;
      int32_t* const at = p.table + slot * p.table_stride + (e - slot * p.max_pages);
      const int32_t id = *at;
      if (id < live || !is_page(p, id)) continue;
      int lo = 0, hi = moved;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (src[mid] < id) lo = mid + 1;
        else hi = mid;
      }
      if (lo < moved && src[lo] == id) *at = free_ids[lo];
    }
  for (int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x; k < moved; k += (int64_t)gridDim.x * 256) {
    p.refs[free_ids[k]] = p.refs[src[k]];
    p.refs[src[k]] = 0;
  }
  const int64_t pieces = pieces_of(p.page_bytes), each = p.layers * pieces;
  for (int64_t item = blockIdx.x; item < moved * each; item += gridDim.x) {
    const int64_t k = item / each, part = item - k * each, layer = part / pieces;
    copy_piece(p, layer, src[k], free_ids[k], part - layer * pieces);
  }
}

// ---------------------------------------------------------------------------------------------- host

int check_pool(const bsg_page_pool* q, bool data, bool table, bool refs) {
  if (!q) return fail(BSG_ERR_ARG, "pool is null");
  if (q->num_pages < 1 || q->num_pages > 0x7fffffff - 8 * kScan) return fail(BSG_ERR_ARG, "pool: num_pages=%lld", (long long)q->num_pages);
  if (data) {
    if (!q->pages || !q->scales) return fail(BSG_ERR_ARG, "pool: null pointer (pages=%p scales=%p)", q->pages, (void*)q->scales);
    if (q->layers < 1 || q->page_bytes < 16 || q->page_bytes % 16 != 0 || q->page_scales < 0)
      return fail(BSG_ERR_ARG, "pool: layers=%lld page_bytes=%lld page_scales=%lld", (long long)q->layers,
                  (long long)q->page_bytes, (long long)q->page_scales);
    if (!is_aligned(q->pages, 16) || !is_aligned(q->scales, 4))
      return fail(BSG_ERR_ALIGN, "pool: pages must be 16-byte and scales 4-byte aligned");
  }
  if (table) {
    if (!q->page_table) return fail(BSG_ERR_ARG, "pool: page_table is null");
    if (q->page_size < 1 || q->num_slots < 1 || q->max_pages < 1 || q->table_stride < q->max_pages)
      return fail(BSG_ERR_ARG, "pool: page_size=%d num_slots=%d max_pages=%d table_stride=%lld", q->page_size,
                  q->num_slots, q->max_pages, (long long)q->table_stride);
    // what append and attention take of a row
    if ((int64_t)q->max_pages * q->page_size > BSG_KV_MAX_TOKENS)
      return fail(BSG_ERR_UNSUPPORTED, "pool: %d pages of %d tokens in a row", q->max_pages, q->page_size);
  }
  if (refs && !q->refcounts) return fail(BSG_ERR_ARG, "pool: refcounts is null");
  return BSG_OK;
}

int check_rows(int32_t n) {
  if (n < 0) return fail(BSG_ERR_ARG, "n=%d", n);
  if (n > BSG_PAGES_MAX_ROWS) return fail(BSG_ERR_UNSUPPORTED, "%d slots in one call (at most %d)", n, BSG_PAGES_MAX_ROWS);
  return BSG_OK;
}

Pool device_pool(const bsg_page_pool* q) {
  Pool p;
  p.pages = (uint8_t*)q->pages;
  p.scales = q->scales;
  p.table = q->page_table;
  p.lengths = q->lengths;
  p.refs = q->refcounts;
  p.layers = q->layers;
  p.page_bytes = q->page_bytes;
  p.page_scales = q->page_scales;
  p.table_stride = q->table_stride;
  p.num_pages = (int32_t)q->num_pages;
  p.page_size = q->page_size;
  p.num_slots = q->num_slots;
  p.max_pages = q->max_pages;
  return p;
}

int check_workspace(const bsg_page_pool* q, const void* ws, int64_t ws_bytes) {
  const int64_t need = bsg_pages_workspace_bytes(q->num_pages);
  if (!ws || ws_bytes < need)
    return fail(BSG_ERR_WORKSPACE, "workspace of %lld bytes, %lld needed", (long long)ws_bytes, (long long)need);
  if (!is_aligned(ws, 16)) return fail(BSG_ERR_ALIGN, "workspace must be 16-byte aligned");
  return BSG_OK;
}

unsigned copy_grid(int64_t items) { return (unsigned)(items < kCopyGroups ? items : kCopyGroups); }

}  // namespace

extern "C" int64_t bsg_pages_workspace_bytes(int64_t num_pages) {
  if (num_pages < 1 || num_pages > 0x7fffffff - 8 * kScan) return -1;
  return kHeader + kRows + ceil_div(num_pages, 4) * 16 * 2;
}

extern "C" int bsg_pages_copy(const bsg_page_pool* pool, const int32_t* src, const int32_t* dst, int32_t n,
                              void* stream) {
  if (const int rc = check_pool(pool, true, false, false)) return rc;
  if (n < 0) return fail(BSG_ERR_ARG, "n=%d", n);
  if (n == 0) return BSG_OK;
  if (!src || !dst) return fail(BSG_ERR_ARG, "null pointer (src=%p dst=%p)", (const void*)src, (const void*)dst);
  hipLaunchKernelGGL(bsg_pages_copy_kernel, dim3(copy_grid(n * pool->layers * pieces_of(pool->page_bytes))), dim3(256), 0, (hipStream_t)stream,
                     device_pool(pool), src, dst, n);
  return launch_status("bsg_pages_copy");
}

extern "C" int bsg_pages_fork(const bsg_page_pool* pool, const int32_t* parents, const int32_t* children, int32_t n,
                              void* stream) {
  if (const int rc = check_pool(pool, false, true, true)) return rc;
  if (const int rc = check_rows(n)) return rc;
  if (!pool->lengths) return fail(BSG_ERR_ARG, "pool: lengths is null");
  if (n == 0) return BSG_OK;
  if (!parents || !children)
    return fail(BSG_ERR_ARG, "null pointer (parents=%p children=%p)", (const void*)parents, (const void*)children);
  const int64_t groups = ceil_div(pool->max_pages, kForkCols) + 1;
  if (groups > kLaunchGroups) return fail(BSG_ERR_UNSUPPORTED, "pool: max_pages=%d", pool->max_pages);
  hipLaunchKernelGGL(bsg_pages_fork_kernel, dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream, device_pool(pool), parents,
                     children, n);
  return launch_status("bsg_pages_fork");
}

extern "C" int bsg_pages_free(const bsg_page_pool* pool, const int32_t* slots, int32_t n, void* stream) {
  if (const int rc = check_pool(pool, false, true, true)) return rc;
  if (const int rc = check_rows(n)) return rc;
  if (!pool->lengths) return fail(BSG_ERR_ARG, "pool: lengths is null");
  if (n == 0) return BSG_OK;
  if (!slots) return fail(BSG_ERR_ARG, "slots is null");
  const int64_t gy = ceil_div(pool->max_pages, 256);
  if (gy > 65535) return fail(BSG_ERR_UNSUPPORTED, "pool: max_pages=%d", pool->max_pages);
  hipLaunchKernelGGL(bsg_pages_free_kernel, dim3((unsigned)n, (unsigned)gy), dim3(256), 0, (hipStream_t)stream,
                     device_pool(pool), slots);
  return launch_status("bsg_pages_free");
}

extern "C" int bsg_pages_extend(const bsg_page_pool* pool, const int32_t* slots, const int32_t* new_tokens, int32_t n,
                                int32_t* served, void* ws, int64_t ws_bytes, void* stream) {
  if (const int rc = check_pool(pool, true, true, true)) return rc;
  if (const int rc = check_rows(n)) return rc;
  if (!pool->lengths) return fail(BSG_ERR_ARG, "pool: lengths is null");
  if (n == 0) return BSG_OK;
  if (!new_tokens || !served)
    return fail(BSG_ERR_ARG, "null pointer (new_tokens=%p served=%p)", (const void*)new_tokens, (void*)served);
  if (!slots && n > pool->num_slots) return fail(BSG_ERR_ARG, "%d rows, %d slots", n, pool->num_slots);
  if (const int rc = check_workspace(pool, ws, ws_bytes)) return rc;
  Row* const rows = (Row*)((uint8_t*)ws + kHeader);
  int32_t* const free_ids = (int32_t*)((uint8_t*)ws + kHeader + kRows);
  const Pool p = device_pool(pool);
  const hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(bsg_pages_extend_plan_kernel, dim3(1), dim3(kScan), 0, st, p, slots, new_tokens, n, served, rows,
                     free_ids);
  // few rows need every piece a work-group of its own; many fill the machine with fewer
  int64_t gy = pool->layers * pieces_of(pool->page_bytes);
  if (gy > ceil_div(4 * kCopyGroups, n)) gy = ceil_div(4 * kCopyGroups, n);
  hipLaunchKernelGGL(bsg_pages_extend_kernel, dim3((unsigned)n, (unsigned)gy), dim3(256), 0, st, p, rows, free_ids);
  return launch_status("bsg_pages_extend");
}

extern "C" int bsg_pages_compact(const bsg_page_pool* pool, int32_t* counts, void* ws, int64_t ws_bytes, void* stream) {
  if (const int rc = check_pool(pool, true, true, true)) return rc;
  if (!counts) return fail(BSG_ERR_ARG, "counts is null");
  if (const int rc = check_workspace(pool, ws, ws_bytes)) return rc;
  int32_t* const header = (int32_t*)ws;
  int32_t* const live_ids = (int32_t*)((uint8_t*)ws + kHeader + kRows);
  int32_t* const free_ids = live_ids + ceil_div(pool->num_pages, 4) * 4;
  const Pool p = device_pool(pool);
  const hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(bsg_pages_compact_plan_kernel, dim3(1), dim3(kScan), 0, st, p, counts, header, live_ids, free_ids);
  hipLaunchKernelGGL(bsg_pages_compact_kernel, dim3((unsigned)kCopyGroups), dim3(256), 0, st, p, header, live_ids,
                     free_ids);
  return launch_status("bsg_pages_compact");
}
