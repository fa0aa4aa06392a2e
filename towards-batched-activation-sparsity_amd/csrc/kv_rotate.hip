// kv_rotate.hip — queries and keys normed by head and rotated by position, and the keys and values quantised into the
// 8-bit paged cache, in one pass (include/bsgdraft.h).
//
// Of a head's D channels x, y = x rsqrt(mean(x^2) + eps) w where there is a norm, and the first R channels turn in
// pairs: (a, b) -> (a cos - b sin, a sin + b cos).  All of it is in 32 bits, of which the queries are rounded to their
// type and the keys to e4m3 once.
//
// Two kinds of work-groups share a launch.  Those of the cache are kv_append.hip's: a wave a 16-token tile of a (page,
// head, keys or values), lane 16 g + t with channels 64 c + 16 g .. +15 of token t, so that a pair's other half lies in the
// lane itself (R = 128: the other c; R = 16: 8 channels on; neighbours), or in lane ^ 32 or ^ 16 (R = 64, 32).  Those of
// the queries take a row of D channels with D / 16 lanes, two runs of 8 channels each, chosen so that a pair's halves meet
// in one lane: eight (D = 128) or sixteen rows a wave.

#include "bsgdraft.h"
#include "draft_tree.hpp"
#include "kv_quant.hpp"

using namespace bsgk;

namespace bsgk {
int check_kv_cache(const bsg_kv_cache* c);
int check_kv_batch(int64_t tokens, int32_t rows, const int32_t* slots, const int32_t* cu, int32_t max_new,
                   const bsg_kv_cache* c, int dtype);
}  // namespace bsgk

namespace {

struct RotateParams {
  const uint16_t* x[2];  // keys, values
  int64_t st[2], sh[2];
  const uint16_t* q;
  uint16_t* out;
  int64_t q_st, q_sh, o_st, o_sh;
  const float* cos;
  const float* sin;
  const uint16_t* q_norm;
  const uint16_t* k_norm;
  const int32_t* turns;    // the position of each token, or null
  const int32_t* parents;  // or a tree, or null
  int64_t turn_stride;
  float eps;
  int32_t turn_count, dims, interleaved;
  uint8_t* pages;
  float* scales;
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* slots;
  const int32_t* cu;
  int64_t table_stride, tokens;
  int32_t num_pages, heads, q_heads, num_slots, max_pages, max_new, pages_per_row, wide;
  int32_t first_unit, units, kv_groups;  // of the cache, in this launch: the first unit, units in all, work-groups
  int32_t first_query, queries, per_row;  // of the queries: waves' worth of rows, of which each sequence has per_row
};

// A sequence of the batch, as a wave sees it.
struct Sequence {
  int64_t from, to, len;
  int slot;
  bool fine;
};
__device__ __forceinline__ Sequence sequence(const RotateParams& p, int row, bool real) {
  Sequence s;
  s.from = (int64_t)row * p.max_new, s.to = s.from + p.max_new;
  s.slot = real ? row : -1;
  if (p.slots && real) s.slot = p.slots[row];
  s.len = s.slot >= 0 && s.slot < p.num_slots ? p.lengths[s.slot] : 0;  // on its way beside the offsets
  if (p.cu && real) s.from = p.cu[row], s.to = p.cu[row + 1];
  s.fine = s.slot >= 0 && s.slot < p.num_slots && s.from >= 0 && s.from < s.to && s.to <= p.tokens;
  return s;
}

// By what position token i of a sequence turns.  All lanes of the wave call it.
__device__ __forceinline__ int64_t turn_of(const RotateParams& p, const Sequence& s, int64_t i, bool on) {
  const int64_t start = s.len - (s.to - s.from);
  if (p.parents) {
    const int lane = threadIdx.x & 63;
    const int64_t n = s.to - s.from < kTreeNodes ? s.to - s.from : kTreeNodes;
    const int depth = depth_of(load_parent(p.parents, s.from, s.fine ? (int)n : 0, lane), lane);
    return start + from_lane(depth, (int)i & 63);
  }
  if (p.turns) return on ? p.turns[s.from + i] : 0;
  return start + i;
}

// Eight 16-bit numbers as 32-bit ones.
template <typename T>
__device__ __forceinline__ void widen8(u32x4 v, float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) f[2 * i] = low_half<T>(v[i]), f[2 * i + 1] = high_half<T>(v[i]);
}
__device__ __forceinline__ u32x4 load8(const uint16_t* at, bool wide) {
  if (wide) return *(const u32x4*)at;
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = at[2 * i] | (uint32_t)at[2 * i + 1] << 16;
  return v;
}
template <typename T>
__device__ __forceinline__ uint32_t narrow(float a, float b);
template <>
__device__ __forceinline__ uint32_t narrow<_Float16>(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
}
template <>
__device__ __forceinline__ uint32_t narrow<__bf16>(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
}

// cos and sin of N consecutive angles of a position; NaN where the table has no such position.
template <int N>
__device__ __forceinline__ void load_turn(const RotateParams& p, int64_t turn, int first, float* c, float* s) {
  const bool there = turn >= 0 && turn < p.turn_count;
  const float nan = __builtin_nanf("");
  const int64_t at = (there ? turn : 0) * p.turn_stride + first;
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    const f32x4 cv = *(const f32x4*)(p.cos + at + 4 * i), sv = *(const f32x4*)(p.sin + at + 4 * i);
#pragma unroll
    for (int j = 0; j < 4; ++j) c[4 * i + j] = there ? cv[j] : nan, s[4 * i + j] = there ? sv[j] : nan;
  }
}
__device__ __forceinline__ void turn_pair(float& a, float& b, float c, float s) {
  const float x = a, y = b;
  a = x * c - y * s, b = x * s + y * c;
}

// A lane's channels 64 c + 16 g .. +15 of a key, turned.  All lanes of the wave call it.
template <int C>
__device__ __forceinline__ void turn_key(const RotateParams& p, int64_t turn, int g, float f[C][16]) {
  const int R = p.dims;
  float c[16], s[16];
  if (p.interleaved) {
#pragma unroll
    for (int k = 0; k < C; ++k) {
      if (64 * k + 16 * g >= R) continue;
      load_turn<8>(p, turn, 32 * k + 8 * g, c, s);
#pragma unroll
      for (int i = 0; i < 8; ++i) turn_pair(f[k][2 * i], f[k][2 * i + 1], c[i], s[i]);
    }
    return;
  }
  if (C == 2 && R == 128) {
    load_turn<16>(p, turn, 16 * g, c, s);
#pragma unroll
    for (int i = 0; i < 16; ++i) turn_pair(f[0][i], f[C - 1][i], c[i], s[i]);
  } else if (R == 16) {
    if (g != 0) return;
    load_turn<8>(p, turn, 0, c, s);
#pragma unroll
    for (int i = 0; i < 8; ++i) turn_pair(f[0][i], f[0][i + 8], c[i], s[i]);
  } else {
    // the other half of a pair is lane ^ 32's (R = 64) or ^ 16's (R = 32) channel
    const bool second = R == 64 ? g >= 2 : g == 1, in = R == 64 || g < 2;
    if (in) load_turn<16>(p, turn, R == 64 ? 16 * (g & 1) : 0, c, s);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float other = R == 64 ? lane_xor<32>(f[0][i]) : lane_xor<16>(f[0][i]);
      if (in) f[0][i] = second ? other * s[i] + f[0][i] * c[i] : f[0][i] * c[i] - other * s[i];
    }
  }
}

// The largest finite magnitude in the wave; only where an infinity is among them are those taken out.
template <int X>
__device__ __forceinline__ float wave_top(float m) {
  m = fmaxf(m, lane_xor<X>(m));
  if constexpr (X > 1) m = wave_top<X / 2>(m);
  return m;
}
template <int C>
__device__ __forceinline__ float finite_top(const float f[C][16]) {
  float m = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i) m = fmaxf(m, __builtin_fabsf(f[c][i]));  // a NaN is no maximum
  m = wave_top<32>(m);
  if (m == __builtin_inff()) {
    m = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float a = __builtin_fabsf(f[c][i]);
        m = a < __builtin_inff() ? fmaxf(m, a) : m;
      }
    m = wave_top<32>(m);
  }
  return m;
}

// A wave's rows of queries.
template <typename T, int D>
__device__ __forceinline__ void turn_queries(const RotateParams& p, uint32_t unit) {
  constexpr int L = D / 16, ROWS = 64 / L;  // lanes of a row, rows of a wave
  const int lane = threadIdx.x & 63, j = lane % L;
  const int row = unit / (uint32_t)p.per_row, nth = unit - row * p.per_row;
  const Sequence s = sequence(p, row, unit < (uint32_t)p.queries);
  const int64_t count = !s.fine ? 0 : s.to - s.from < p.max_new ? s.to - s.from : p.max_new;
  const uint32_t r = nth * ROWS + lane / L, i = r / (uint32_t)p.q_heads;
  const int head = r - i * p.q_heads;
  const bool on = i < count;
  if (!__any(on)) return;
  const int64_t turn = turn_of(p, s, i, on);
  if (!on) return;
  const int R = p.dims;
  int lo, hi, first;
  if (p.interleaved) lo = 16 * j, hi = lo + 8, first = 8 * j;
  else if (16 * j < R) lo = 8 * j, hi = lo + R / 2, first = lo;
  else lo = 16 * j, hi = lo + 8, first = 0;
  const uint16_t* const src = p.q + (s.from + i) * p.q_st + (int64_t)head * p.q_sh;
  float a[8], b[8];
  widen8<T>(*(const u32x4*)(src + lo), a);
  widen8<T>(*(const u32x4*)(src + hi), b);
  float c[8], sn[8];
  if (16 * j < R) load_turn<8>(p, turn, first, c, sn);
  if (p.q_norm) {
    float w[8], z[8];
    widen8<T>(*(const u32x4*)(p.q_norm + lo), w);
    widen8<T>(*(const u32x4*)(p.q_norm + hi), z);
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += a[k] * a[k] + b[k] * b[k];
    sum += lane_xor<1>(sum);  // a row's lanes are on together
    sum += lane_xor<2>(sum);
    if constexpr (L == 8) sum += lane_xor<4>(sum);
    const float by = __builtin_amdgcn_rsqf(sum * (1.f / D) + p.eps);
#pragma unroll
    for (int k = 0; k < 8; ++k) a[k] = a[k] * by * w[k], b[k] = b[k] * by * z[k];
  }
  if (16 * j < R) {
    if (p.interleaved) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        turn_pair(a[2 * k], a[2 * k + 1], c[k], sn[k]);
        turn_pair(b[2 * k], b[2 * k + 1], c[k + 4], sn[k + 4]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) turn_pair(a[k], b[k], c[k], sn[k]);
    }
  }
  uint16_t* const dst = p.out + (s.from + i) * p.o_st + (int64_t)head * p.o_sh;
  u32x4 y, z;
#pragma unroll
  for (int k = 0; k < 4; ++k) y[k] = narrow<T>(a[2 * k], a[2 * k + 1]), z[k] = narrow<T>(b[2 * k], b[2 * k + 1]);
  *(u32x4*)(dst + lo) = y;
  *(u32x4*)(dst + hi) = z;
}

template <typename T, int D, int P>
__global__ __launch_bounds__(P <= 64 ? 256 : 512) void bsg_kv_append_rotated_kernel(RotateParams p) {
  constexpr int THREADS = P <= 64 ? 256 : 512;
  constexpr int W = P / 16;                   // waves of a page
  constexpr int UNITS = P <= 64 ? 4 / W : 1;  // (page, head, K/V) units of a work-group
  constexpr int C = D / 64;
  __shared__ float s_max[UNITS][W];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if ((int)blockIdx.x >= p.kv_groups) {
    turn_queries<T, D>(p, p.first_query + (blockIdx.x - p.kv_groups) * (THREADS / 64) + wave);
    return;
  }
  const int unit = wave / W, tile = wave % W;
  // units in the order head, K/V, page of the row, row: neighbours write neighbouring bytes
  const uint32_t u = p.first_unit + blockIdx.x * UNITS + unit, per_page = 2 * p.heads;
  const uint32_t rp = u / per_page, hk = u - rp * per_page;
  const int head = hk >> 1, kv = hk & 1;
  const int row = rp / p.pages_per_row, nth = rp - row * p.pages_per_row;

  const Sequence s = sequence(p, row, u < (uint32_t)p.units);
  bool fine = s.fine;
  const int64_t start = s.len - (s.to - s.from);  // may be below 0: tokens at negative positions are not written
  const int64_t most = (int64_t)p.max_pages * P;
  int64_t end = s.to - s.from > p.max_new ? start + p.max_new : s.len;  // of the tokens that are written
  if (end > most) end = most;
  const int64_t j = (start > 0 ? start : 0) / P + nth;
  const int64_t lo = start > j * P ? start - j * P : 0;   // first new token of the page
  const int64_t hi = end < (j + 1) * P ? end - j * P : P;  // end of its tokens
  fine = fine && lo < hi && j < p.max_pages;
  int32_t page = -1;
  if (fine) page = p.table[(int64_t)s.slot * p.table_stride + j];

  const int t = lane & 15, g = lane >> 4;
  const int tok = tile * 16 + t;
  const bool is_new = fine && tok >= lo && tok < hi;
  const int64_t nth_new = j * P + tok - start;  // of the sequence's new tokens
  float f[C][16];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i) f[c][i] = 0.f;
  if (is_new) {
    const uint16_t* src = p.x[kv] + (s.from + nth_new) * p.st[kv] + (int64_t)head * p.sh[kv] + 16 * g;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i) widen8<T>(load8(src + 64 * c + 8 * i, p.wide), f[c] + 8 * i);
  }
  if (kv == 0) {
    const int64_t turn = turn_of(p, s, is_new ? nth_new : 0, is_new);
    if (p.k_norm) {
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += f[c][i] * f[c][i];
      sum += lane_xor<16>(sum);
      sum += lane_xor<32>(sum);
      const float by = __builtin_amdgcn_rsqf(sum * (1.f / D) + p.eps);
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float w[8];
          widen8<T>(*(const u32x4*)(p.k_norm + 64 * c + 16 * g + 8 * i), w);
#pragma unroll
          for (int k = 0; k < 8; ++k) f[c][8 * i + k] = f[c][8 * i + k] * by * w[k];
        }
    }
    turn_key<C>(p, is_new ? turn : 0, g, f);
    if (!is_new) {  // no token: 0 x inf may have made a NaN of it
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) f[c][i] = 0.f;
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
  float a = finite_top<C>(f);
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
      y[c][i] = to_e4m3(f[c][4 * i] * inv, f[c][4 * i + 1] * inv, f[c][4 * i + 2] * inv, f[c][4 * i + 3] * inv);
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

// Of one launch: multiples of a work-group's units and waves, and with up to 512 threads each within what a launch
// takes.  A batch without a bound on its sequences' new tokens has every sequence take as many pages and rows as all
// tokens fill.
constexpr int64_t kLaunchUnits = 1 << 21;

template <typename T, int D>
void launch(RotateParams p, int page_size, int64_t queries, hipStream_t st) {
  const int per = page_size <= 64 ? 64 / page_size : 1;  // units of a work-group
  const int waves = page_size <= 64 ? 4 : 8;
  for (int64_t unit = 0, query = 0; unit < p.units || query < queries;) {
    const int64_t units = p.units - unit < kLaunchUnits ? p.units - unit : kLaunchUnits;
    const int64_t more = queries - query < kLaunchUnits ? queries - query : kLaunchUnits;
    p.first_unit = (int32_t)unit;
    p.kv_groups = (int32_t)ceil_div(units, per);
    p.first_query = (int32_t)query;
    const dim3 grid((unsigned)(p.kv_groups + ceil_div(more, waves)));
    switch (page_size) {
      case 16: hipLaunchKernelGGL((bsg_kv_append_rotated_kernel<T, D, 16>), grid, dim3(256), 0, st, p); break;
      case 32: hipLaunchKernelGGL((bsg_kv_append_rotated_kernel<T, D, 32>), grid, dim3(256), 0, st, p); break;
      case 64: hipLaunchKernelGGL((bsg_kv_append_rotated_kernel<T, D, 64>), grid, dim3(256), 0, st, p); break;
      default: hipLaunchKernelGGL((bsg_kv_append_rotated_kernel<T, D, 128>), grid, dim3(512), 0, st, p); break;
    }
    unit += units, query += more;
  }
}

int check_rotary(const bsg_rotary* r, const bsg_kv_cache* c, int32_t max_new) {
  if (!r) return fail(BSG_ERR_ARG, "rotary is null");
  if (!r->cos || !r->sin) return fail(BSG_ERR_ARG, "rotary: null pointer (cos=%p sin=%p)", (const void*)r->cos, (const void*)r->sin);
  if (r->dims != 16 && r->dims != 32 && r->dims != 64 && r->dims != 128)
    return fail(BSG_ERR_UNSUPPORTED, "rotary: dims=%d (16, 32, 64 or 128)", r->dims);
  if (r->dims > c->head_dim) return fail(BSG_ERR_ARG, "rotary: dims=%d of head_dim=%d", r->dims, c->head_dim);
  if (r->positions < 1 || (r->positions > 1 && r->stride < r->dims / 2))
    return fail(BSG_ERR_ARG, "rotary: positions=%d stride=%lld", r->positions, (long long)r->stride);
  if (!(r->eps >= 0.f) || !(r->eps < __builtin_inff())) return fail(BSG_ERR_ARG, "rotary: eps=%g", r->eps);
  if (!is_aligned(r->cos, 16) || !is_aligned(r->sin, 16) || (r->stride & 3) != 0)
    return fail(BSG_ERR_ALIGN, "rotary: rows of cos and sin must be 16-byte aligned (stride %lld)", (long long)r->stride);
  if (!is_aligned(r->q_norm, 16) || !is_aligned(r->k_norm, 16)) return fail(BSG_ERR_ALIGN, "rotary: norms must be 16-byte aligned");
  if (r->token_positions && r->parents) return fail(BSG_ERR_ARG, "rotary: positions or a tree, not both");
  if (r->parents && max_new > BSG_TREE_NODES)
    return fail(BSG_ERR_UNSUPPORTED, "%d nodes in a tree (at most %d)", max_new, BSG_TREE_NODES);
  return BSG_OK;
}

}  // namespace

extern "C" int bsg_kv_append_rotated(const void* q, int64_t q_stride_t, int64_t q_stride_h, int32_t q_heads, void* out,
                                     int64_t o_stride_t, int64_t o_stride_h, const void* k, int64_t k_stride_t,
                                     int64_t k_stride_h, const void* v, int64_t v_stride_t, int64_t v_stride_h,
                                     int64_t tokens, const bsg_rotary* rotary, const bsg_kv_cache* cache,
                                     const int32_t* slots, int32_t rows, const int32_t* cu, int32_t max_new, int dtype,
                                     void* stream) {
  if (const int rc = check_kv_cache(cache)) return rc;
  if (const int rc = check_kv_batch(tokens, rows, slots, cu, max_new, cache, dtype)) return rc;
  if (const int rc = check_rotary(rotary, cache, max_new)) return rc;
  if (q_heads < 1 || q_heads > 65535) return fail(BSG_ERR_ARG, "q_heads=%d", q_heads);
  if (tokens == 0 || rows == 0 || max_new == 0) return BSG_OK;
  if (!q || !out || !k || !v) return fail(BSG_ERR_ARG, "null pointer (q=%p out=%p k=%p v=%p)", q, out, k, v);
  if (!is_aligned(q, 16) || !is_aligned(out, 16) || ((q_stride_t | q_stride_h | o_stride_t | o_stride_h) & 7) != 0)
    return fail(BSG_ERR_ALIGN, "rows of q and out must be 16-byte aligned (strides %lld, %lld and %lld, %lld)",
                (long long)q_stride_t, (long long)q_stride_h, (long long)o_stride_t, (long long)o_stride_h);
  if (!is_aligned(k, 2) || !is_aligned(v, 2)) return fail(BSG_ERR_ALIGN, "k and v must be 2-byte aligned");
  const int P = cache->page_size;
  const int64_t per_row = ((int64_t)max_new + P - 2) / P + 1;  // pages that max_new tokens can touch
  const int64_t units = per_row * rows * cache->n_heads * 2;
  const int64_t q_row = ceil_div((int64_t)max_new * q_heads * (cache->head_dim / 16), 64), queries = q_row * rows;
  if (units > 0x7fffffff - kLaunchUnits || queries > 0x7fffffff - kLaunchUnits)
    return fail(BSG_ERR_UNSUPPORTED, "%lld tiles of work", (long long)(units > queries ? units : queries));
  if ((int64_t)max_new * q_heads > 0x7fffffff - 64) return fail(BSG_ERR_UNSUPPORTED, "%d tokens x %d heads", max_new, q_heads);
  RotateParams p;
  p.x[0] = (const uint16_t*)k, p.x[1] = (const uint16_t*)v;
  p.st[0] = k_stride_t, p.st[1] = v_stride_t, p.sh[0] = k_stride_h, p.sh[1] = v_stride_h;
  p.q = (const uint16_t*)q, p.out = (uint16_t*)out;
  p.q_st = q_stride_t, p.q_sh = q_stride_h, p.o_st = o_stride_t, p.o_sh = o_stride_h;
  p.cos = rotary->cos, p.sin = rotary->sin;
  p.q_norm = (const uint16_t*)rotary->q_norm, p.k_norm = (const uint16_t*)rotary->k_norm;
  p.turns = rotary->token_positions, p.parents = rotary->parents;
  p.turn_stride = rotary->stride;
  p.eps = rotary->eps;
  p.turn_count = rotary->positions, p.dims = rotary->dims, p.interleaved = rotary->interleaved != 0;
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
  p.q_heads = q_heads;
  p.num_slots = cache->num_slots;
  p.max_pages = cache->max_pages;
  p.max_new = max_new;
  p.pages_per_row = (int32_t)per_row;
  p.units = (int32_t)units;
  p.queries = (int32_t)queries;
  p.per_row = (int32_t)q_row;
  p.wide = is_aligned(k, 16) && is_aligned(v, 16) &&
           ((k_stride_t | k_stride_h | v_stride_t | v_stride_h) & 7) == 0;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == BSG_F16)
    cache->head_dim == 64 ? launch<_Float16, 64>(p, P, queries, st) : launch<_Float16, 128>(p, P, queries, st);
  else
    cache->head_dim == 64 ? launch<__bf16, 64>(p, P, queries, st) : launch<__bf16, 128>(p, P, queries, st);
  return launch_status("bsg_kv_append_rotated");
}
