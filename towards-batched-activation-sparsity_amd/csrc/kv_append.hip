// kv_append.hip — new keys and values into the 8-bit paged cache (include/bsgserve.h).
//
// One wave owns one 16-token tile of a (page, head, keys or values); the page_size / 16 waves of a
// page meet once in LDS, for the largest magnitude.  Lane 16 g + t of a tile holds channels
// 64 c + 16 g .. +15 of token t, two 16-byte loads per c.  For the keys its quantised 16 bytes are
// the lane's 16 bytes of the tile; for the values the four lanes of a quad exchange their 4 x 4
// bytes (tokens x channels), after which each holds dwords of four tokens of one channel, and the
// four rows of 16 lanes their 4 x 4 dwords, after which these too are the lane's 16 bytes.
//
// A wave a tile, and not a page, because a page of 128 tokens would be eight tiles one after the other,
// and because one new token of 64 sequences x 32 heads is 4096 waves as it is.  4 x 2000 tokens x 8 heads of
// 128, bf16, pages of 64 (31 MB in, 16 out): 10.9 us, 4.3 TB/s, bound by HBM.  64 x 1 token x 32 heads, fp16, pages of
// 16: 6.8 us, a chain of three dependent loads from cold caches (length, page, what the page holds) between
// launch and store.

#include "serve.hpp"

using namespace bsgk;

namespace {

struct AppendParams {
  const uint16_t* x[2];  // keys, values
  int64_t st[2], sh[2];
  uint8_t* pages;
  float* scales;
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* slots;
  const int32_t* cu;
  int64_t table_stride, tokens;
  int32_t num_pages, heads, num_slots, max_pages, max_new, pages_per_row, first_unit, units, wide;
};

// Bytes b of the four dwords a quad's lanes hold, to lane b of the quad: the 4 x 4 byte transpose.
__device__ __forceinline__ uint32_t quad_transpose(uint32_t w, int i) {
  const uint32_t w0 = __builtin_amdgcn_mov_dpp(w, 0x00, 0xf, 0xf, true);
  const uint32_t w1 = __builtin_amdgcn_mov_dpp(w, 0x55, 0xf, 0xf, true);
  const uint32_t w2 = __builtin_amdgcn_mov_dpp(w, 0xaa, 0xf, 0xf, true);
  const uint32_t w3 = __builtin_amdgcn_mov_dpp(w, 0xff, 0xf, 0xf, true);
  const uint32_t sel = (uint32_t)i * 0x0101u + 0x0400u;  // byte i of each of two words
  const uint32_t lo = __builtin_amdgcn_perm(w1, w0, sel) & 0xffffu;
  const uint32_t hi = __builtin_amdgcn_perm(w3, w2, sel) & 0xffffu;
  return lo | (hi << 16);
}

// The 4 x 4 transpose of four dwords over the four rows of 16 lanes.
__device__ __forceinline__ void row_transpose(uint32_t w[4]) {
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const auto r = __builtin_amdgcn_permlane32_swap(w[n], w[n + 2], false, false);
    w[n] = r[0], w[n + 2] = r[1];
  }
#pragma unroll
  for (int n = 0; n < 4; n += 2) {
    const auto r = __builtin_amdgcn_permlane16_swap(w[n], w[n + 1], false, false);
    w[n] = r[0], w[n + 1] = r[1];
  }
}

// x / scale to e4m3, rounded to nearest even: the product with a power of two is exact, infinities
// become the largest value, NaN stays.
__device__ __forceinline__ float in_range(float x) { return x != x ? x : fminf(fmaxf(x, -448.f), 448.f); }

__device__ __forceinline__ uint32_t to_e4m3(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(in_range(a), in_range(b), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(in_range(c), in_range(d), r, true);
}

// Four cached numbers under a new, larger scale.
__device__ __forceinline__ uint32_t rescale(uint32_t w, float ratio) {
  return to_e4m3(__builtin_amdgcn_cvt_f32_fp8((int)w, 0) * ratio, __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * ratio,
                 __builtin_amdgcn_cvt_f32_fp8((int)w, 2) * ratio, __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * ratio);
}

// The largest finite magnitude in the wave.  Magnitudes of either 16-bit type order as their bits do; only where
// infinities or NaN are among them are those taken out.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
template <typename T>
constexpr uint32_t kInfBits = 0x7c00u;
template <>
constexpr uint32_t kInfBits<__bf16> = 0x7f80u;

template <int X>
__device__ __forceinline__ u16x2 wave_max(u16x2 m) {
  m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, lane_xor<X>(__builtin_bit_cast(uint32_t, m))));
  if constexpr (X > 1) m = wave_max<X / 2>(m);
  return m;
}
template <typename T, int C>
__device__ __forceinline__ float largest_magnitude(const uint32_t x[C][8]) {
  u16x2 m = {0, 0};
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, x[c][i] & 0x7fff7fffu));
  m = wave_max<32>(m);
  uint32_t top = m.x > m.y ? m.x : m.y;
  if (top >= kInfBits<T>) {
    m = u16x2{0, 0};
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t w = x[c][i] & 0x7fff7fffu;
        const uint32_t lo = w & 0xffffu, hi = w >> 16;
        m = __builtin_elementwise_max(m, u16x2{(unsigned short)(lo < kInfBits<T> ? lo : 0u), (unsigned short)(hi < kInfBits<T> ? hi : 0u)});
      }
    m = wave_max<32>(m);
    top = m.x > m.y ? m.x : m.y;
  }
  return low_half<T>(top);
}

// The least power of two s in [2^-40, 2^80] with a <= 448 s, from the bits of a = 1.m x 2^e:
// 448 = 1.75 x 2^8.
__device__ __forceinline__ float scale_for(float a) {
  const int e = (int)((__builtin_bit_cast(uint32_t, a) + 0x1fffffu) >> 23) - 127 - 8;
  const int c = e < BSG_KV_SCALE_MIN_EXP ? BSG_KV_SCALE_MIN_EXP : e > BSG_KV_SCALE_MAX_EXP ? BSG_KV_SCALE_MAX_EXP : e;
  return __builtin_bit_cast(float, (uint32_t)(c + 127) << 23);
}

template <typename T, int D, int P>
__global__ __launch_bounds__(P <= 64 ? 256 : 512) void bsg_kv_append_kernel(AppendParams p) {
  constexpr int W = P / 16;                // waves of a page
  constexpr int UNITS = P <= 64 ? 4 / W : 1;  // (page, head, K/V) units of a work-group
  constexpr int C = D / 64;
  __shared__ float s_max[UNITS][W];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int unit = wave / W, tile = wave % W;
  // units in the order head, K/V, page of the row, row: neighbours write neighbouring bytes
  const uint32_t u = p.first_unit + blockIdx.x * UNITS + unit, per_page = 2 * p.heads;
  const uint32_t rp = u / per_page, hk = u - rp * per_page;
  const int head = hk >> 1, kv = hk & 1;
  const int row = rp / p.pages_per_row, nth = rp - row * p.pages_per_row;

  const bool real = u < (uint32_t)p.units;
  int64_t from = (int64_t)row * p.max_new, to = from + p.max_new;
  int slot = real ? row : -1;
  if (p.slots && real) slot = p.slots[row];
  const int64_t len = slot >= 0 && slot < p.num_slots ? p.lengths[slot] : 0;  // on its way beside the offsets
  if (p.cu && real) from = p.cu[row], to = p.cu[row + 1];
  bool fine = slot >= 0 && slot < p.num_slots && from >= 0 && from < to && to <= p.tokens;
  const int64_t start = len - (to - from);  // may be below 0: tokens at negative positions are not written
  const int64_t most = (int64_t)p.max_pages * P;
  int64_t end = to - from > p.max_new ? start + p.max_new : len;  // of the tokens that are written
  if (end > most) end = most;
  const int64_t j = (start > 0 ? start : 0) / P + nth;
  const int64_t lo = start > j * P ? start - j * P : 0;                 // first new token of the page
  const int64_t hi = end < (j + 1) * P ? end - j * P : P;               // end of its tokens
  fine = fine && lo < hi && j < p.max_pages;
  int32_t page = -1;
  if (fine) page = p.table[(int64_t)slot * p.table_stride + j];

  const int t = lane & 15, g = lane >> 4;
  const int tok = tile * 16 + t;
  const bool is_new = fine && tok >= lo && tok < hi;
  uint32_t x[C][8];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) x[c][i] = 0;
  if (is_new) {
    const uint16_t* src = p.x[kv] + (from + (j * P + tok - start)) * p.st[kv] + (int64_t)head * p.sh[kv] + 16 * g;
    if (p.wide) {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const u32x4 v = *(const u32x4*)(src + 64 * c + 8 * i);
          x[c][4 * i] = v.x, x[c][4 * i + 1] = v.y, x[c][4 * i + 2] = v.z, x[c][4 * i + 3] = v.w;
        }
    } else {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[c][i] = src[64 * c + 2 * i] | (uint32_t)src[64 * c + 2 * i + 1] << 16;
    }
  }
  // The new numbers were asked for beside the page; what the page decides comes now.
  fine = fine && page >= 0 && page < p.num_pages;
  float* const scale_at = p.scales + ((int64_t)page * p.heads + head) * 2 + kv;
  const float old = fine && lo > 0 ? *scale_at : 0.f;
  uint8_t* const dst = p.pages + (((int64_t)page * p.heads + head) * 2 + kv) * (P * D) + (int64_t)tile * 16 * D;
  // Bytes of the values' dwords (tokens 4q .. 4q+3) that are new, and that hold earlier tokens; what
  // is there is on its way while the new ones are weighed.
  uint32_t fresh = 0, held = 0;
  u32x4 was[C];
  const int v_off = (t >> 2) * 256 + (4 * g + (t & 3)) * 16;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const int k = tile * 16 + (t & 12) + b;
    if (k >= lo && k < hi) fresh |= 0xffu << (8 * b);
    if (k < lo) held |= 0xffu << (8 * b);
  }
#pragma unroll
  for (int c = 0; c < C; ++c) {
    was[c] = u32x4{0u, 0u, 0u, 0u};
    if (kv == 1 && fine && fresh != 0xffffffffu && (fresh | held) != 0) was[c] = *(const u32x4*)(dst + c * 1024 + v_off);
  }
  float a = largest_magnitude<T, C>(x);
  if constexpr (W > 1) {  // also: every wave has the old scale before one writes the new
    if (lane == 0) s_max[unit][tile] = a;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) a = fmaxf(a, s_max[unit][i]);
  }
  if (!fine) return;

  float scale = scale_for(a), ratio = 1.f;
  if (lo > 0) {
    if (old >= scale) scale = old;
    ratio = old / scale;
  }
  if (tile == 0 && lane == 0) *scale_at = scale;
  // what this wave's tile does not have to write: no new token, and no earlier one to round again
  if (tile * 16 >= hi || (tile * 16 + 16 <= lo && ratio == 1.f)) return;

  const float inv = 1.f / scale;
  uint32_t y[C][4];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      y[c][i] = to_e4m3(low_half<T>(x[c][2 * i]) * inv, high_half<T>(x[c][2 * i]) * inv,
                        low_half<T>(x[c][2 * i + 1]) * inv, high_half<T>(x[c][2 * i + 1]) * inv);
  if (kv == 0) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      u32x4* const at = (u32x4*)(dst + c * 1024 + lane * 16);
      if (is_new) {
        *at = u32x4{y[c][0], y[c][1], y[c][2], y[c][3]};
      } else if (tok < lo && ratio != 1.f) {
        const u32x4 v = *at;
        *at = u32x4{rescale(v.x, ratio), rescale(v.y, ratio), rescale(v.z, ratio), rescale(v.w, ratio)};
      }
    }
  } else {
    const bool rounds = held != 0 && ratio != 1.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      uint32_t w[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) w[n] = quad_transpose(y[c][n], t & 3);
      row_transpose(w);  // lane 16 g + 4 q + i: channels 16 n + 4 g + i of tokens 4 q .. 4 q + 3
      u32x4* const at = (u32x4*)(dst + c * 1024 + v_off);
      u32x4 v = {w[0], w[1], w[2], w[3]};
      if (fresh != 0xffffffffu) {
        if (fresh == 0 && !rounds) continue;
        u32x4 kept = was[c];
        if (rounds)
          kept = (u32x4{rescale(kept.x, ratio), rescale(kept.y, ratio), rescale(kept.z, ratio), rescale(kept.w, ratio)} & held) |
                 (kept & ~held);
        v = (v & fresh) | (kept & ~fresh);
      }
      *at = v;
    }
  }
}

// Of one launch: a multiple of a work-group's units, and with up to 512 threads each within what a launch takes.  A
// batch without a bound on its sequences' new tokens has every sequence take as many pages as all tokens fill.
constexpr int64_t kLaunchUnits = 1 << 22;

template <typename T, int D>
void launch(AppendParams p, int page_size, hipStream_t st) {
  for (int64_t first = 0; first < p.units; first += kLaunchUnits) {
    const int64_t units = p.units - first < kLaunchUnits ? p.units - first : kLaunchUnits;
    const auto grid = [&](int per) { return dim3((unsigned)ceil_div(units, per)); };
    p.first_unit = (int32_t)first;
    switch (page_size) {
      case 16: hipLaunchKernelGGL((bsg_kv_append_kernel<T, D, 16>), grid(4), dim3(256), 0, st, p); break;
      case 32: hipLaunchKernelGGL((bsg_kv_append_kernel<T, D, 32>), grid(2), dim3(256), 0, st, p); break;
      case 64: hipLaunchKernelGGL((bsg_kv_append_kernel<T, D, 64>), grid(1), dim3(256), 0, st, p); break;
      default: hipLaunchKernelGGL((bsg_kv_append_kernel<T, D, 128>), grid(1), dim3(512), 0, st, p); break;
    }
  }
}

}  // namespace

namespace bsgk {

int check_kv_cache(const bsg_kv_cache* c) {
  if (!c) return fail(BSG_ERR_ARG, "cache is null");
  if (!c->pages || !c->scales || !c->page_table || !c->lengths)
    return fail(BSG_ERR_ARG, "cache: null pointer (pages=%p scales=%p page_table=%p lengths=%p)", c->pages,
                (const void*)c->scales, (const void*)c->page_table, (const void*)c->lengths);
  if (c->num_pages < 1 || c->num_pages > 0x7fffffff || c->n_heads < 1 || c->n_heads > 65535 || c->num_slots < 1 ||
      c->max_pages < 1 || c->table_stride < c->max_pages)
    return fail(BSG_ERR_ARG, "cache: num_pages=%lld n_heads=%d num_slots=%d max_pages=%d table_stride=%lld",
                (long long)c->num_pages, c->n_heads, c->num_slots, c->max_pages, (long long)c->table_stride);
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
    return fail(BSG_ERR_UNSUPPORTED, "cache: page_size=%d (16, 32, 64 or 128)", c->page_size);
  if (c->head_dim != 64 && c->head_dim != 128)
    return fail(BSG_ERR_UNSUPPORTED, "cache: head_dim=%d (64 or 128)", c->head_dim);
  if (!is_aligned(c->pages, 16) || !is_aligned(c->scales, 8))
    return fail(BSG_ERR_ALIGN, "cache: pages must be 16-byte and scales 8-byte aligned");
  // the attention's positions are 32-bit and go past a row's end by up to 4096
  if ((int64_t)c->max_pages * c->page_size > BSG_KV_MAX_TOKENS)
    return fail(BSG_ERR_UNSUPPORTED, "cache: %d pages of %d tokens in a row", c->max_pages, c->page_size);
  return BSG_OK;
}

int check_kv_batch(int64_t tokens, int32_t rows, const int32_t* slots, const int32_t* cu, int32_t max_new,
                   const bsg_kv_cache* c, int dtype) {
  if (dtype != BSG_F16 && dtype != BSG_BF16) return fail(BSG_ERR_DTYPE, "dtype=%d (0=fp16, 1=bf16)", dtype);
  if (tokens < 0 || rows < 0 || max_new < 0 || tokens > 0x7fffffff)
    return fail(BSG_ERR_ARG, "tokens=%lld rows=%d max_new=%d", (long long)tokens, rows, max_new);
  if (!cu && tokens != (int64_t)rows * max_new)
    return fail(BSG_ERR_ARG, "without cu, tokens=%lld must be rows x max_new = %lld", (long long)tokens,
                (long long)rows * max_new);
  if (!slots && rows > c->num_slots)
    return fail(BSG_ERR_ARG, "%d rows, %d slots", rows, c->num_slots);
  return BSG_OK;
}

}  // namespace bsgk

extern "C" int bsg_kv_append(const void* k, int64_t k_stride_t, int64_t k_stride_h, const void* v, int64_t v_stride_t,
                             int64_t v_stride_h, int64_t tokens, const bsg_kv_cache* cache, const int32_t* slots,
                             int32_t rows, const int32_t* cu, int32_t max_new, int dtype, void* stream) {
  if (const int rc = check_kv_cache(cache)) return rc;
  if (const int rc = check_kv_batch(tokens, rows, slots, cu, max_new, cache, dtype)) return rc;
  if (tokens == 0 || rows == 0 || max_new == 0) return BSG_OK;
  if (!k || !v) return fail(BSG_ERR_ARG, "null pointer (k=%p v=%p)", k, v);
  if (!is_aligned(k, 2) || !is_aligned(v, 2)) return fail(BSG_ERR_ALIGN, "k and v must be 2-byte aligned");
  const int P = cache->page_size;
  const int64_t per_row = ((int64_t)max_new + P - 2) / P + 1;  // pages that max_new tokens can touch
  const int64_t units = per_row * rows * cache->n_heads * 2;
  if (units > 0x7fffffff) return fail(BSG_ERR_UNSUPPORTED, "%lld tiles of work", (long long)units);
  AppendParams p;
  p.x[0] = (const uint16_t*)k, p.x[1] = (const uint16_t*)v;
  p.st[0] = k_stride_t, p.st[1] = v_stride_t, p.sh[0] = k_stride_h, p.sh[1] = v_stride_h;
  p.pages = (uint8_t*)cache->pages;
  p.scales = cache->scales;
  p.table = cache->page_table;
  p.lengths = cache->lengths;
  p.slots = slots;
  p.cu = cu;
  p.table_stride = cache->table_stride;
  p.tokens = tokens;
  p.num_pages = (int32_t)cache->num_pages;
  p.heads = cache->n_heads;
  p.num_slots = cache->num_slots;
  p.max_pages = cache->max_pages;
  p.max_new = max_new;
  p.pages_per_row = (int32_t)per_row;
  p.units = (int32_t)units;
  p.wide = is_aligned(k, 16) && is_aligned(v, 16) &&
           ((k_stride_t | k_stride_h | v_stride_t | v_stride_h) & 7) == 0;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == BSG_F16)
    cache->head_dim == 64 ? launch<_Float16, 64>(p, P, st) : launch<_Float16, 128>(p, P, st);
  else
    cache->head_dim == 64 ? launch<__bf16, 64>(p, P, st) : launch<__bf16, 128>(p, P, st);
  return launch_status("bsg_kv_append");
}
