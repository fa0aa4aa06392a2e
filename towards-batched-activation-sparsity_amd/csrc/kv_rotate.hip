// kv_rotate.hip — queries and keys normed by head and rotated by position, and the keys and values quantised into the
// 8-bit paged cache, in one pass (include/bsgdraft.h).
//
// Of a head's D channels x, y = x rsqrt(mean(x^2) + eps) w where there is a norm, and the first R channels turn in
// pairs: (a, b) -> (a cos - b sin, a sin + b cos).  All of it is in 32 bits, of which the queries are rounded to their
// type and the keys to e4m3 once.
//
// Two kinds of work-groups share a launch.  Those of the cache are much like kv_append.hip's: a wave a 16-token tile of a (page,
// head), keys and values, lane 16 g + t with channels 64 c + 16 g .. +15 of token t, so that a pair's other half lies in the
// lane itself (R = 128: the other c; R = 16: 8 channels on; neighbours), or in lane ^ 32 or ^ 16 (R = 64, 32).  Those of
// the queries take a row of D channels with D / 16 lanes, two runs of 8 channels each, chosen so that a pair's halves meet
// in one lane: eight (D = 128) or sixteen rows at a time, kRows times, with one load of a token's angles for the rows that share it.

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

// Lane j: how deep node j of a sequence lies in its tree.  All lanes of the wave call it.
__device__ __forceinline__ int depths(const RotateParams& p, const Sequence& s) {
  const int lane = threadIdx.x & 63;
  const int64_t n = s.to - s.from < kTreeNodes ? s.to - s.from : kTreeNodes;
  return depth_of(load_parent(p.parents, s.from, s.fine ? (int)n : 0, lane), lane);
}
// By what position token i of a sequence turns.  All lanes of the wave call it.
__device__ __forceinline__ int64_t turn_of(const RotateParams& p, const Sequence& s, int64_t i, bool on, int depth) {
  const int64_t start = s.len - (s.to - s.from);
  if (p.parents) return start + from_lane(depth, (int)i & 63);
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

// cos and sin of eight angles of a position; NaN where the table has no such position.  Asked for in one place and looked
// at in another, so that they are on their way beside what is turned.
struct Angles {
  f32x4 c[2], s[2];
  bool there;
  __device__ __forceinline__ void ask(const RotateParams& p, int64_t turn, int first) {
    there = turn >= 0 && turn < p.turn_count;
    const int64_t at = (there ? turn : 0) * p.turn_stride + first;
#pragma unroll
    for (int i = 0; i < 2; ++i) c[i] = *(const f32x4*)(p.cos + at + 4 * i), s[i] = *(const f32x4*)(p.sin + at + 4 * i);
  }
  __device__ __forceinline__ float cos(int i) const { return there ? c[i / 4][i % 4] : __builtin_nanf(""); }
  __device__ __forceinline__ float sin(int i) const { return there ? s[i / 4][i % 4] : __builtin_nanf(""); }
};
__device__ __forceinline__ void turn_pair(float& a, float& b, float c, float s) {
  const float x = a, y = b;
  a = x * c - y * s, b = x * s + y * c;
}

// A lane's channels 64 c + 16 g .. +15 of a key are turned by twice eight angles, the H-th of which key_angles names; they come
// one after the other, for the registers (a wave more on each SIMD).  All lanes of the wave call it.
__device__ __forceinline__ int key_angles(const RotateParams& p, int g, int H) {
  const int R = p.dims, at = p.interleaved ? 8 * g + 32 * H : (R == 128 ? 16 * g : R == 64 ? 16 * (g & 1) : 0) + 8 * H;
  return at < R / 2 ? at : 0;  // of channels that are not turned: any
}
template <int C, int H>
__device__ __forceinline__ void turn_key(const RotateParams& p, const Angles& a, int g, float f[C][16]) {
  const int R = p.dims;
  if (p.interleaved) {
    if (H < C && 64 * H + 16 * g < R) {
#pragma unroll
      for (int i = 0; i < 8; ++i) turn_pair(f[H < C ? H : 0][2 * i], f[H < C ? H : 0][2 * i + 1], a.cos(i), a.sin(i));
    }
  } else if (C == 2 && R == 128) {
#pragma unroll
    for (int i = 0; i < 8; ++i) turn_pair(f[0][8 * H + i], f[C - 1][8 * H + i], a.cos(i), a.sin(i));
  } else if (R == 16) {
    if (H != 0 || g != 0) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) turn_pair(f[0][i], f[0][i + 8], a.cos(i), a.sin(i));
  } else {
    // the other half of a pair is lane ^ 32's (R = 64) or ^ 16's (R = 32) channel
    const bool second = R == 64 ? g >= 2 : g == 1, in = R == 64 || g < 2;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float& x = f[0][8 * H + i];
      const float other = R == 64 ? lane_xor<32>(x) : lane_xor<16>(x);
      if (in) x = second ? other * a.sin(i) + x * a.cos(i) : x * a.cos(i) - other * a.sin(i);
    }
  }
}

// The largest finite magnitude in the wave, and whether all of its numbers are finite.  Only where they are not are the
// others looked at one by one.
template <int X>
__device__ __forceinline__ float wave_top(float m) {
  m = fmaxf(m, lane_xor<X>(m));
  if constexpr (X > 1) m = wave_top<X / 2>(m);
  return m;
}
template <int C>
__device__ __forceinline__ float finite_top(const float f[C][16], bool* finite) {
  float m = 0.f, none = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i) m = fmaxf(m, __builtin_fabsf(f[c][i])), none = __builtin_fmaf(f[c][i], 0.f, none);
  m = wave_top<32>(m);
  *finite = !__any(none != 0.f);  // an infinity or NaN times 0 is NaN
  if (!*finite) {
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

// A wave's rows of queries: kRows times as many as its lanes hold, since rows of one token, which follow each other, share
// their angles and all share the norm.  1, 2, 4 times: 45, 41, 44 us for 6000 tokens x 32 heads (with their keys and values, each
// of which had a wave of its own then).
constexpr int kRows = 2;
template <typename T, int D>
__device__ __forceinline__ void turn_queries(const RotateParams& p, uint32_t unit) {
  constexpr int L = D / 16, ROWS = 64 / L;  // lanes of a row, rows of a wave at a time
  const int lane = threadIdx.x & 63, j = lane % L;
  const int row = unit / (uint32_t)p.per_row, nth = unit - row * p.per_row;
  const Sequence s = sequence(p, row, unit < (uint32_t)p.queries);
  const int64_t count = !s.fine ? 0 : s.to - s.from < p.max_new ? s.to - s.from : p.max_new;
  const uint32_t first_row = nth * (kRows * ROWS);
  if ((int64_t)first_row >= count * p.q_heads) return;
  const int R = p.dims;
  int lo, hi, first;
  if (p.interleaved) lo = 16 * j, hi = lo + 8, first = 16 * j < R ? 8 * j : 0;
  else if (16 * j < R) lo = 8 * j, hi = lo + R / 2, first = lo;
  else lo = 16 * j, hi = lo + 8, first = 0;
  uint32_t tok[kRows];
  u32x4 v[kRows][2];
  int64_t to[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const uint32_t r = first_row + i * ROWS + lane / L;
    tok[i] = r / (uint32_t)p.q_heads;
    const int head = r - tok[i] * p.q_heads;
    const int64_t t = s.from + (tok[i] < count ? tok[i] : 0);  // rows past the last one read the first
    const uint16_t* const src = p.q + t * p.q_st + (int64_t)head * p.q_sh;
    v[i][0] = *(const u32x4*)(src + lo), v[i][1] = *(const u32x4*)(src + hi);
    to[i] = t * p.o_st + (int64_t)head * p.o_sh;
  }
  u32x4 norm[2] = {{0u, 0u, 0u, 0u}, {0u, 0u, 0u, 0u}};
  if (p.q_norm) norm[0] = *(const u32x4*)(p.q_norm + lo), norm[1] = *(const u32x4*)(p.q_norm + hi);
  const int depth = p.parents ? depths(p, s) : 0;
  Angles angles;
  angles.ask(p, turn_of(p, s, tok[0], tok[0] < count, depth), first);
  float w[16];
  widen8<T>(norm[0], w);
  widen8<T>(norm[1], w + 8);
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const bool on = tok[i] < count;
    if (i > 0) {
      const int64_t turn = turn_of(p, s, tok[i], on, depth);
      if (tok[i] != tok[i - 1]) angles.ask(p, turn, first);
    }
    float a[8], b[8];
    widen8<T>(v[i][0], a);
    widen8<T>(v[i][1], b);
    if (p.q_norm) {
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += a[k] * a[k] + b[k] * b[k];
      sum += lane_xor<1>(sum);
      sum += lane_xor<2>(sum);
      if constexpr (L == 8) sum += lane_xor<4>(sum);
      const float by = __builtin_amdgcn_rsqf(sum * (1.f / D) + p.eps);
#pragma unroll
      for (int k = 0; k < 8; ++k) a[k] = a[k] * by * w[k], b[k] = b[k] * by * w[k + 8];
    }
    if (16 * j < R) {
      if (p.interleaved) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          turn_pair(a[2 * k], a[2 * k + 1], angles.cos(k), angles.sin(k));
          turn_pair(b[2 * k], b[2 * k + 1], angles.cos(k + 4), angles.sin(k + 4));
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) turn_pair(a[k], b[k], angles.cos(k), angles.sin(k));
      }
    }
    u32x4 y, z;
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = narrow<T>(a[2 * k], a[2 * k + 1]), z[k] = narrow<T>(b[2 * k], b[2 * k + 1]);
    if (on) {
      *(u32x4*)(p.out + to[i] + lo) = y;
      *(u32x4*)(p.out + to[i] + hi) = z;
    }
  }
}

// To e4m3, of numbers that are finite and within 448, or of any.
__device__ __forceinline__ uint32_t quantise(float a, float b, float c, float d, bool plain) {
  if (!plain) return to_e4m3(a, b, c, d);
  const int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

// A page's new scale for the largest magnitude of its new numbers, and its old one over that.
struct Scale {
  float now, ratio;
};
__device__ __forceinline__ Scale scale_of(float top, float old, bool holds) {
  Scale s = {scale_for(top), 1.f};
  if (holds) {
    if (old >= s.now) s.now = old;
    s.ratio = old / s.now;
  }
  return s;
}

// HBM bounds it: 6000 tokens of prompts, 32 heads on 8, norms (175 MB): 37 us, 4.7 TB/s.  What is on its way counts: keys and values in
// one wave (in one each: 45), four waves a SIMD by halves of the angles (64 trees of up to 16 nodes, 32 heads: 15.3 us; all angles
// at once 18).  One token is a chain of three loads, 6 us.  Keys in 64 bits, so that none is rounded to the neighbour of
// what its exact value would be (of some 10^7 about 10 are): 47 and 23 us.
template <typename T, int D, int P>
__global__ __launch_bounds__(P <= 64 ? 256 : 512) void bsg_kv_append_rotated_kernel(RotateParams p) {
  constexpr int THREADS = P <= 64 ? 256 : 512;
  constexpr int W = P / 16;                   // waves of a page
  constexpr int UNITS = P <= 64 ? 4 / W : 1;  // (page, head) units of a work-group
  constexpr int C = D / 64;
  __shared__ f32x2 s_max[UNITS][W];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if ((int)blockIdx.x >= p.kv_groups) {
    turn_queries<T, D>(p, p.first_query + (blockIdx.x - p.kv_groups) * (THREADS / 64) + wave);
    return;
  }
  const int unit = wave / W, tile = wave % W;
  // units in the order head, page of the row, row: neighbours write neighbouring bytes
  const uint32_t u = p.first_unit + blockIdx.x * UNITS + unit;
  const uint32_t rp = u / (uint32_t)p.heads;
  const int head = u - rp * p.heads;
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
  const int64_t nth_new = is_new ? j * P + tok - start : 0;  // of the sequence's new tokens; lanes without one read the first
  u32x4 raw[C][2];
  uint32_t v[C][8];
  Angles angles;
  int64_t turn = 0;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[c][i] = 0;
  if (fine) {
    const uint16_t* const k_src = p.x[0] + (s.from + nth_new) * p.st[0] + (int64_t)head * p.sh[0] + 16 * g;
    const uint16_t* const v_src = p.x[1] + (s.from + nth_new) * p.st[1] + (int64_t)head * p.sh[1] + 16 * g;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i) raw[c][i] = load8(k_src + 64 * c + 8 * i, p.wide);
    if (!p.parents) turn = turn_of(p, s, nth_new, is_new, 0), angles.ask(p, turn, key_angles(p, g, 0));
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const u32x4 x = load8(v_src + 64 * c + 8 * i, p.wide);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[c][4 * i + e] = is_new ? x[e] : 0u;
      }
    if (p.parents) turn = turn_of(p, s, nth_new, is_new, depths(p, s)), angles.ask(p, turn, key_angles(p, g, 0));
  }
  // The new numbers were asked for beside the page; what the page decides comes now, and is on its way while the new
  // ones are turned and weighed.
  fine = fine && page >= 0 && page < p.num_pages;
  const int64_t block = ((int64_t)page * p.heads + head) * 2;
  const f32x2 old = fine && lo > 0 ? *(const f32x2*)(p.scales + block) : f32x2{0.f, 0.f};
  uint8_t* const k_dst = p.pages + block * (P * D) + (int64_t)tile * 16 * D;
  uint8_t* const v_dst = k_dst + P * D;
  // bytes of the values' dwords (tokens 4q .. 4q+3) that are new, and that hold earlier tokens
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
    if (fine && fresh != 0xffffffffu && (fresh | held) != 0) was[c] = *(const u32x4*)(v_dst + c * 1024 + v_off);
  }

  float f[C][16];
  const bool any_new = __any(is_new);
  if (any_new) {
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i) widen8<T>(raw[c][i], f[c] + 8 * i);
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
          widen8<T>(*(const u32x4*)(p.k_norm + 64 * c + 16 * g + 8 * i), w);  // in every cache: not held till here
#pragma unroll
          for (int k = 0; k < 8; ++k) f[c][8 * i + k] = f[c][8 * i + k] * by * w[k];
        }
    }
    turn_key<C, 0>(p, angles, g, f);
    angles.ask(p, turn, key_angles(p, g, 1));
    turn_key<C, 1>(p, angles, g, f);
  }
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i) f[c][i] = is_new ? f[c][i] : 0.f;
  bool finite;
  f32x2 top = {finite_top<C>(f, &finite), largest_magnitude<T, C>(v)};
  if constexpr (W > 1) {  // also: every wave has the old scales before one writes the new
    if (lane == 0) s_max[unit][tile] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) top.x = fmaxf(top.x, s_max[unit][i].x), top.y = fmaxf(top.y, s_max[unit][i].y);
  }
  if (!fine) return;

  const Scale ks = scale_of(top.x, old.x, lo > 0), vs = scale_of(top.y, old.y, lo > 0);
  if (tile == 0 && lane == 0) *(f32x2*)(p.scales + block) = f32x2{ks.now, vs.now};
  if (tile * 16 >= hi) return;  // none of this wave's tokens is there

  // keys: no new one, and no earlier one to round again, leaves the tile as it is
  if (tile * 16 + 16 > lo || ks.ratio != 1.f) {
    const float inv = 1.f / ks.now;
    const bool plain = finite && top.x * inv <= 448.f;  // which may fail where the scale is at its limit
#pragma unroll
    for (int c = 0; c < C; ++c) {
      u32x4* const at = (u32x4*)(k_dst + c * 1024 + lane * 16);
      if (is_new) {
        u32x4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          y[i] = quantise(f[c][4 * i] * inv, f[c][4 * i + 1] * inv, f[c][4 * i + 2] * inv, f[c][4 * i + 3] * inv, plain);
        *at = y;
      } else if (tok < lo && ks.ratio != 1.f) {
        const u32x4 x = *at;
        *at = u32x4{rescale(x.x, ks.ratio), rescale(x.y, ks.ratio), rescale(x.z, ks.ratio), rescale(x.w, ks.ratio)};
      }
    }
  }
  if (tile * 16 + 16 > lo || vs.ratio != 1.f) {
    const float inv = 1.f / vs.now, ratio = vs.ratio;
    const bool rounds = held != 0 && ratio != 1.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = quad_transpose(to_e4m3(low_half<T>(v[c][2 * i]) * inv, high_half<T>(v[c][2 * i]) * inv, low_half<T>(v[c][2 * i + 1]) * inv,
                                      high_half<T>(v[c][2 * i + 1]) * inv), t & 3);
      row_transpose(w);  // lane 16 g + 4 q + i: channels 16 n + 4 g + i of tokens 4 q .. 4 q + 3
      u32x4* const at = (u32x4*)(v_dst + c * 1024 + v_off);
      u32x4 y = {w[0], w[1], w[2], w[3]};
      if (fresh != 0xffffffffu) {
        if (fresh == 0 && !rounds) continue;
        u32x4 kept = was[c];
        if (rounds)
          kept = (u32x4{rescale(kept.x, ratio), rescale(kept.y, ratio), rescale(kept.z, ratio), rescale(kept.w, ratio)} & held) |
                 (kept & ~held);
        y = (y & fresh) | (kept & ~fresh);
      }
      *at = y;
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
  const int64_t units = per_row * rows * cache->n_heads;
  const int64_t q_row = ceil_div((int64_t)max_new * q_heads * (cache->head_dim / 16), 64 * kRows), queries = q_row * rows;
  if (units > 0x7fffffff - kLaunchUnits || queries > 0x7fffffff - kLaunchUnits)
    return fail(BSG_ERR_UNSUPPORTED, "%lld tiles of work", (long long)(units > queries ? units : queries));
  if ((int64_t)max_new * q_heads > 0x7fffffff - 64 * kRows) return fail(BSG_ERR_UNSUPPORTED, "%d tokens x %d heads", max_new, q_heads);
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
