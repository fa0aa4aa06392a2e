// kv_attention.hpp — the kernels of attention over the 8-bit paged cache: of tokens that follow each other
// (include/bsgserve.h, kv_attention.hip), and of drafted ones that form a tree (include/bsgdraft.h, kv_tree.hip).
//
// Per cached head, the rows of a call are its new tokens x the query heads that share it.  With
// every product transposed, S^T = K Q^T and O^T = V^T P^T, a cache tile of 16 tokens is the A
// operand of v_mfma_f32_16x16x32 as it lies in memory, 16 query rows are its columns, and the
// accumulator layout of S^T (column = row of the call, four consecutive tokens per lane) is the B
// operand that O^T needs: nothing is shuffled between the two products.
//
// Scales and softmax in one exponent: with s2 = log2(e) sm_scale ks (q . k8) and lv = log2(vs), the weight of a
// token is w = 2^(s2 + lv - B), where B = M - 13 for a maximum M of s2 + lv that a later one may pass by an octave or
// more, so that O = sum w v8 / sum w / vs whatever B is.  w stays within fp16, as which it goes to the matrix
// unit: every weight down to 2^-27 of the largest keeps 11 bits.  Its sum is taken in fp32 before.
// From 2^22 octaves on s2 + lv and M - 13 are rounded by octaves themselves, so there B = M, and the difference is
// taken between rounded sums, which is exact near the maximum.
#pragma once

#include <utility>

#include "draft_tree.hpp"
#include "serve.hpp"

using namespace bsgk;

namespace bsgk {
int check_kv_cache(const bsg_kv_cache* c);
int check_kv_batch(int64_t tokens, int32_t rows, const int32_t* slots, const int32_t* cu, int32_t max_new,
                   const bsg_kv_cache* c, int dtype);
}  // namespace bsgk

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxSplits = 32;    // parts of one row
constexpr float kShift = 13.f;  // weights go up to 2^(kShift + kSlack), within fp16
constexpr float kFarScore = 0x1p22f;  // octaves from which on a score's last bit is half an octave or more
// Octaves within which score and base may come in one step, rounded once: against a base that was made from rounded scores a weight is
// then off by up to half a score's last bit, 2^-13 octaves here, a quarter of what its rounding to fp16 takes (at 2^21 it would be 9%).
constexpr float kNearScore = 0x1p11f;
constexpr float kSlack = 1.5f;  // octaves by which, in the first kernel, a score may exceed the running maximum before that moves
constexpr float kMostWeight = 65504.f;  // of fp16; four weights at the maximum make half of it

struct AttnParams {
  const uint16_t* q;
  uint16_t* out;
  float* lse;
  const uint8_t* pages;
  const float* scales;
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* slots;
  const int32_t* cu;
  float* part;         // [tile of rows][split][rows][D + 2]
  uint32_t* counters;  // [tile of rows]
  int64_t q_st, q_sh, o_st, o_sh, table_stride, tokens;
  float scale2;        // sm_scale * log2(e)
  int32_t num_pages, kv_heads, group, num_slots, max_pages, page_shift, max_new, row_tiles, splits, chunk;
  const int32_t* parents;  // of a tree's nodes
};

template <typename T>
struct Elem;
template <>
struct Elem<_Float16> {
  typedef f16x8 x8;
  static __device__ __forceinline__ uint32_t word(uint32_t w, bool high) {
    return __builtin_bit_cast(uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true)
                                             : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false));
  }
  static __device__ __forceinline__ f32x4 mfma(x8 a, x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
  }
};
template <>
struct Elem<__bf16> {
  typedef bf16x8 x8;
  static __device__ __forceinline__ uint32_t word(uint32_t w, bool high) {
    return __builtin_bit_cast(uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true)
                                             : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false));
  }
  static __device__ __forceinline__ f32x4 mfma(x8 a, x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
  }
};

// Eight e4m3 numbers as 16-bit ones (exact in either type).
template <typename T>
__device__ __forceinline__ typename Elem<T>::x8 widen(uint32_t lo, uint32_t hi) {
  return __builtin_bit_cast(typename Elem<T>::x8, u32x4{Elem<T>::word(lo, false), Elem<T>::word(lo, true),
                                                        Elem<T>::word(hi, false), Elem<T>::word(hi, true)});
}

// The base B for a maximum, both in octaves.
__device__ __forceinline__ float base_of(float m) { return __builtin_fabsf(m) < kFarScore ? m - kShift : m; }

// Over the four lanes that hold one column: lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float column_max(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v);
  const auto x = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  v = fmaxf(as_float(x[0]), as_float(x[1]));
  const uint32_t c = __builtin_bit_cast(uint32_t, v);
  const auto y = __builtin_amdgcn_permlane16_swap(c, c, false, false);
  return fmaxf(as_float(y[0]), as_float(y[1]));
}
__device__ __forceinline__ float column_sum(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v);
  const auto x = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  v = as_float(x[0]) + as_float(x[1]);
  const uint32_t c = __builtin_bit_cast(uint32_t, v);
  const auto y = __builtin_amdgcn_permlane16_swap(c, c, false, false);
  return as_float(y[0]) + as_float(y[1]);
}

// The bytes of four consecutive tokens of which the first n exist.
__device__ __forceinline__ uint32_t byte_mask(int n) {
  return n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << (8 * n)) - 1u;
}
// 0x38 (1.0 in e4m3) in each byte that is NaN (0x7f or 0xff).
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  const uint32_t x = (w & 0x7f7f7f7fu) + 0x01010101u;  // bit 7 of a byte: all seven bits were set
  return ((x & 0x80808080u) >> 7) * 0x38u;
}

// What one row sees: the tokens before `until`, or with a tree those before `first` and of the 64 from there on the
// ones in `mask`.
template <bool TREE>
struct Sight {
  int until;
  static __device__ __forceinline__ Sight none() { return Sight{0}; }
  __device__ __forceinline__ bool operator()(int t) const { return t < until; }
};
template <>
struct Sight<true> {
  int first;
  uint64_t mask;
  static __device__ __forceinline__ Sight none() { return Sight{-64, 0}; }
  __device__ __forceinline__ bool operator()(int t) const {
    const int d = t - first;
    return d < 0 || (d < 64 && (mask >> d & 1) != 0);
  }
  // of the tokens t .. t + 3, as bits
  __device__ __forceinline__ uint32_t four(int t) const {
    const int d = t - first;
    if (d >= 0) return d < 64 ? (uint32_t)(mask >> d) & 15u : 0u;
    return d <= -4 ? 15u : ((uint32_t)mask << -d | ((1u << -d) - 1u)) & 15u;
  }
};

// A NaN among values that some rows do not see: the matrix unit would spread it to all rows (0 x
// NaN), so it goes to those that see it by a product of flags, and leaves the values.  v: four tiles of 16 channels
// of two 16-token tiles, t: the lane's first token, acc: their four accumulators of each 16 rows.
template <int RT, bool TREE>
__device__ __forceinline__ void nan_values(u32x4 v[2], int t, const Sight<TREE>* sees, f32x4* acc, int stride) {
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    uint32_t f[4];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        f[2 * a + j] = Elem<_Float16>::pack(sees[i](t + 16 * a + 2 * j) ? 1.f : 0.f, sees[i](t + 16 * a + 2 * j + 1) ? 1.f : 0.f);
    const f16x8 flags = __builtin_bit_cast(f16x8, u32x4{f[0], f[1], f[2], f[3]});
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      f32x4 n = {0.f, 0.f, 0.f, 0.f};
      n = Elem<_Float16>::mfma(widen<_Float16>(nan_bytes(v[0][d]), nan_bytes(v[1][d])), flags, n);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n[j] > 0.f) acc[i * stride + d][j] = __builtin_nanf("");
    }
  }
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const uint32_t n = nan_bytes(v[a][d]);  // 0x38 to 0xff
      v[a][d] &= ~(n | (n << 1) | (n << 2) | (n >> 1) | (n >> 2) | (n >> 3));
    }
}

// A work-group of four waves computes RT x 16 rows of one cached head of one sequence over one chunk
// of its tokens; wave w takes the 32-token steps w, w + 4, ..., each with its own running maximum, and the
// waves meet in LDS at the end.  Chunks meet in the workspace: the last one to arrive sums them in order.
//
// Steps are interleaved over the waves, so that a work-group reads on as one stream; a step of a wave is
// 8 KiB (D = 128), straight into registers in the order the matrix unit wants, and one more is on its
// way, which with two work-groups on a compute unit covers HBM's latency.  64 sequences of up to 4096 tokens x 32
// heads of 128, fp16 (1.44 GB): 232 us, 6.2 TB/s.  64 x 4 new tokens over 1500: 84 us (5.8 TB/s); 5 x 32 heads over
// 60001 tokens of 8 cached heads, bf16: 81 us (5.5 TB/s): bound by HBM, past the rate of a copy
// (5.0).  One sequence of 777 tokens: 8.9 us, the chain length, page, scale and tile, then the parts' meeting.
template <typename T, int D, int RT, bool TREE>
__global__ __launch_bounds__(256, 2) void bsg_kv_attention_kernel(AttnParams p) {
  constexpr int C = D / 64, DT = D / 16, ROWS = 16 * RT, LD = D + 4;
  typedef typename Elem<T>::x8 x8;
  __shared__ float s_acc[ROWS * LD];
  __shared__ float s_m[4][ROWS], s_l[4][ROWS];
  __shared__ uint32_t s_last;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 15, g = lane >> 4;
  const int head = blockIdx.x / p.row_tiles, rt = blockIdx.x - head * p.row_tiles;
  const int split = blockIdx.y, row = blockIdx.z;

  const int slot = p.slots ? p.slots[row] : row;
  int64_t from = (int64_t)row * p.max_new, to = from + p.max_new;
  if (p.cu) from = p.cu[row], to = p.cu[row + 1];
  if (from < 0 || to > p.tokens || from >= to) return;
  const int count = (int)(to - from < p.max_new ? to - from : p.max_new);
  const int rows = count * p.group - rt * ROWS;  // rows of this tile that exist (at most ROWS count)
  if (rows <= 0) return;
  int len = slot >= 0 && slot < p.num_slots ? p.lengths[slot] : 0;
  const int most = p.max_pages << p.page_shift;
  len = len < 0 ? 0 : len > most ? most : len;
  const int first = len - (int)(to - from);  // position of the first new token (below 0: it sees nothing)

  // tokens that the tile's rows see: row r is new token r / group
  const int r_last = rt * ROWS + (rows < ROWS ? rows : ROWS) - 1;
  int end = first + r_last / p.group + 1;
  end = end < 0 ? 0 : end;
  // tokens that every row sees
  const int all_see = TREE ? (first < 0 ? 0 : first) : first + rt * ROWS / p.group + 1;
  const int chunks = end <= p.chunk ? 1 : (end + p.chunk - 1) / p.chunk < p.splits ? (end + p.chunk - 1) / p.chunk : p.splits;
  if (split >= chunks) return;
  const int t_begin = split * p.chunk;
  const int t_end = split == chunks - 1 ? end : t_begin + p.chunk;

  // Q^T as the B operand: column = row of the tile, channels in the order the keys' tiles have them
  x8 qf[RT][2 * C];
  Sight<TREE> sees[RT];
  uint64_t lineage = 0;  // lane j: node j and its ancestors
  if constexpr (TREE) lineage = lineage_of(load_parent(p.parents, from, count, lane), lane);
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int r = rt * ROWS + 16 * i + col;
    const int tok = r / p.group, h = r - tok * p.group;
    const bool on = 16 * i + col < rows;
    if constexpr (TREE) {
      const uint64_t mask = from_lane(lineage, tok & 63);
      sees[i] = on ? Sight<true>{first, mask} : Sight<true>::none();
    } else {
      sees[i] = on ? Sight<false>{first + tok + 1} : Sight<false>::none();
    }
#pragma unroll
    for (int c = 0; c < 2 * C; ++c) {
      u32x4 v = {0u, 0u, 0u, 0u};
      if (on)
        v = *(const u32x4*)(p.q + (from + tok) * p.q_st + (int64_t)(head * p.group + h) * p.q_sh + 64 * (c >> 1) +
                            16 * g + 8 * (c & 1));
      qf[i][c] = __builtin_bit_cast(x8, v);
    }
  }

  f32x4 acc[RT][DT];
  float base[RT], l[RT];  // -inf: no token seen
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    base[i] = -__builtin_inff(), l[i] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[i][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const int32_t* const table = p.table + (int64_t)(slot < 0 || slot >= p.num_slots ? 0 : slot) * p.table_stride;
  const int64_t head_bytes = (int64_t)2 * D << p.page_shift;
  const int in_page = (1 << p.page_shift) - 1;
  const uint8_t* const mine = p.pages + lane * 16;
  struct Step {
    u32x4 k[2][C], v[2][C];
  };
  // Up to 32 steps (64 tiles) of the wave at a time: lane j keeps the page and scales of its tile j,
  // from where they come as scalars; the step after the one at work is on its way.
  for (int b0 = t_begin + 32 * wave; b0 < t_end; b0 += 32 * 128) {
    const int steps = (t_end - b0 + 127) / 128 < 32 ? (t_end - b0 + 127) / 128 : 32;
    int lane_page = -1;
    f32x2 lane_scale = {0.f, 0.f};
    {
      const int t = b0 + 128 * (lane >> 1) + 16 * (lane & 1);
      if (t < t_end) {
        const int page = table[t >> p.page_shift];
        if (page >= 0 && page < p.num_pages) {
          lane_page = page;
          lane_scale = *(const f32x2*)(p.scales + 2 * ((int64_t)page * p.kv_heads + head));
        }
      }
    }
    const auto fetch = [&](int n, Step& s) {
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const int t = b0 + 128 * n + 16 * a;
        const int page = __builtin_amdgcn_readlane(lane_page, 2 * n + a);
        const uint8_t* const at =
            mine + ((int64_t)(page < 0 ? 0 : page) * p.kv_heads + head) * head_bytes + (int64_t)((t & in_page) * D);
#pragma unroll
        for (int c = 0; c < C; ++c) {
          s.k[a][c] = __builtin_nontemporal_load((const u32x4*)(at + c * 1024));
          s.v[a][c] = __builtin_nontemporal_load((const u32x4*)(at + (head_bytes >> 1) + c * 1024));
        }
      }
    };
    float lane_ks = 0.f, lane_lv = 0.f, lane_iv = 0.f;
    const auto take = [&](int n, Step& s) {
      const int t0 = b0 + 128 * n;
      auto& kr = s.k;
      auto& vr = s.v;
      float ks[2], lv[2], iv[2];
      bool there[2];
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        there[a] = __builtin_amdgcn_readlane(lane_page, 2 * n + a) >= 0;
        ks[a] = as_float(__builtin_amdgcn_readlane(__builtin_bit_cast(int, lane_ks), 2 * n + a));
        lv[a] = as_float(__builtin_amdgcn_readlane(__builtin_bit_cast(int, lane_lv), 2 * n + a));
        iv[a] = as_float(__builtin_amdgcn_readlane(__builtin_bit_cast(int, lane_iv), 2 * n + a));
      }
      const bool partial = t0 + 32 > all_see || !there[0] || !there[1];
      uint32_t nan = 0;
      if (partial) {
        // tokens past the tile's end may be anything
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          const uint32_t mask = there[a] ? byte_mask(t_end - (t0 + 16 * a + 4 * g)) : 0u;
#pragma unroll
          for (int c = 0; c < C; ++c) {
            vr[a][c] &= mask;
            nan |= nan_bytes(vr[a][c].x) | nan_bytes(vr[a][c].y) | nan_bytes(vr[a][c].z) | nan_bytes(vr[a][c].w);
          }
        }
      }
      const bool some_nan = partial && __any(nan != 0);

      f16x8 pf[RT];
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        f32x4 s[2];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          s[a] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < C; ++c) {
            s[a] = Elem<T>::mfma(widen<T>(kr[a][c].x, kr[a][c].y), qf[i][2 * c], s[a]);
            s[a] = Elem<T>::mfma(widen<T>(kr[a][c].z, kr[a][c].w), qf[i][2 * c + 1], s[a]);
          }
          uint32_t four = 0;
          if constexpr (TREE) {
            if (partial) four = sees[i].four(t0 + 16 * a + 4 * g);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            s[a][j] = s[a][j] * ks[a] + lv[a];
            if constexpr (TREE) {
              if (partial && (!there[a] || (four >> j & 1u) == 0)) s[a][j] = -__builtin_inff();
            } else {
              if (partial && (!there[a] || t0 + 16 * a + 4 * g + j >= sees[i].until)) s[a][j] = -__builtin_inff();
            }
          }
        }
        float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                         fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        mx = column_max(mx);
        if (__any(mx - base[i] > kShift + kSlack)) {
          const float next = fmaxf(base[i], base_of(mx));
          const float alpha = next == base[i] ? 1.f : __builtin_amdgcn_exp2f(base[i] - next);
          l[i] *= alpha;
#pragma unroll
          for (int d = 0; d < DT; ++d) acc[i][d] *= alpha;
          base[i] = next;
        }
        const float from = base[i] == -__builtin_inff() ? 0.f : base[i];
        float w[2][4];
        uint32_t pw[4];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
#pragma unroll
          for (int j = 0; j < 4; ++j) w[a][j] = __builtin_amdgcn_exp2f(s[a][j] - from);
          pw[2 * a] = Elem<_Float16>::pack(w[a][0], w[a][1]), pw[2 * a + 1] = Elem<_Float16>::pack(w[a][2], w[a][3]);
          l[i] = __builtin_fmaf((w[a][0] + w[a][1]) + (w[a][2] + w[a][3]), iv[a], l[i]);
        }
        pf[i] = __builtin_bit_cast(f16x8, u32x4{pw[0], pw[1], pw[2], pw[3]});
      }
      if (some_nan) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
          u32x4 v[2] = {vr[0][c], vr[1][c]};
          nan_values<RT, TREE>(v, t0 + 4 * g, sees, &acc[0][4 * c], DT);
          vr[0][c] = v[0], vr[1][c] = v[1];
        }
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const f16x8 v = widen<_Float16>(vr[0][d >> 2][d & 3], vr[1][d >> 2][d & 3]);
#pragma unroll
        for (int i = 0; i < RT; ++i) acc[i][d] = Elem<_Float16>::mfma(v, pf[i], acc[i][d]);
      }
    };
    Step even, odd;
    fetch(0, even);
    // the scales were asked for before the step, and are only looked at now
    const float lane_vs = fmaxf(lane_scale.y, 0x1p-100f);
    lane_ks = lane_scale.x * p.scale2, lane_lv = __builtin_amdgcn_logf(lane_vs), lane_iv = __builtin_amdgcn_rcpf(lane_vs);
    for (int n = 0; n < steps; n += 2) {
      if (n + 1 < steps) fetch(n + 1, odd);
      take(n, even);
      if (n + 1 >= steps) break;
      if (n + 2 < steps) fetch(n + 2, even);
      take(n + 1, odd);
    }
  }

  // the waves' parts under a common base
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    l[i] = column_sum(l[i]);
    if (g == 0) s_m[wave][16 * i + col] = base[i], s_l[wave][16 * i + col] = l[i];
  }
  __syncthreads();
  float f[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int r = 16 * i + col;
    const float top = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
    f[i] = base[i] == top ? 1.f : __builtin_amdgcn_exp2f(base[i] - top);
  }
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (wave == w) {
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          f32x4* const at = (f32x4*)(s_acc + (16 * i + col) * LD + 16 * d + 4 * g);
          f32x4 v = acc[i][d] * f[i];
          if (w > 0) v += *at;
          *at = v;
        }
    }
    __syncthreads();
  }

  const int used = rows < ROWS ? rows : ROWS;
  const float* parts = nullptr;
  if (chunks > 1) {
    const int64_t tile = ((int64_t)row * p.kv_heads + head) * p.row_tiles + rt;
    constexpr int PART = ROWS * (D + 2);
    float* const part = p.part + (tile * p.splits + split) * PART;
    parts = p.part + tile * p.splits * PART;
    const __amdgpu_buffer_rsrc_t mine_rsrc = hand_buffer(part, PART * 4);
    for (int e = threadIdx.x; e < used * (D / 4); e += 256) {
      const int r = e / (D / 4), d = (e - r * (D / 4)) * 4;
      hand_store16(mine_rsrc, e * 16, *(const f32x4*)(s_acc + r * LD + d));
    }
    if ((int)threadIdx.x < used) {
      const int r = threadIdx.x;
      const float top = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) sum += s_l[w][r] * (s_m[w][r] == top ? 1.f : __builtin_amdgcn_exp2f(s_m[w][r] - top));
      hand_store((uint64_t*)(part + ROWS * D) + r, __builtin_bit_cast(uint64_t, f32x2{top, sum}));
    }
    hand_publish();
    __syncthreads();
    if (threadIdx.x == 0) s_last = hand_arrive(p.counters + tile) == (uint32_t)(chunks - 1);
    __syncthreads();
    if (!s_last) return;
    if (threadIdx.x == 0) hand_reset(p.counters + tile);
  }

  for (int e = threadIdx.x; e < used * (D / 4); e += 256) {
    const int r = e / (D / 4), d = e % (D / 4) * 4;
    float top = -__builtin_inff(), sum = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    if (chunks > 1) {
      // four numbers of a row from every part, with the part's maximum and sum, eight parts in flight
      constexpr int PART = ROWS * (D + 2), BATCH = 8;
      const __amdgpu_buffer_rsrc_t all = hand_buffer(parts, chunks * PART * 4);
      for (int s = 0; s < chunks; s += BATCH) {
        f32x4 v[BATCH];
        f32x2 ml[BATCH];
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
          const int at = s + j < chunks ? (s + j) * PART * 4 : 0x40000000;  // past the buffer: zeros
          v[j] = hand_load16(all, at + e * 16);
          ml[j] = hand_load8(all, at + (ROWS * D + 2 * r) * 4);
        }
        float high = top;
#pragma unroll
        for (int j = 0; j < BATCH; ++j) high = s + j < chunks ? fmaxf(high, ml[j].x) : high;
        const float f = top == high ? 1.f : __builtin_amdgcn_exp2f(top - high);
        o *= f, sum *= f, top = high;
#pragma unroll
        for (int j = 0; j < BATCH; ++j)
          if (s + j < chunks) {
            const float w = ml[j].x == top ? 1.f : __builtin_amdgcn_exp2f(ml[j].x - top);
            o += v[j] * w, sum += ml[j].y * w;
          }
      }
    } else {
      top = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
#pragma unroll
      for (int w = 0; w < 4; ++w) sum += s_l[w][r] * (s_m[w][r] == top ? 1.f : __builtin_amdgcn_exp2f(s_m[w][r] - top));
      o = *(const f32x4*)(s_acc + r * LD + d);
    }
    const int rr = rt * ROWS + r, tok = rr / p.group, h = head * p.group + rr - tok * p.group;
    const bool nothing = sum == 0.f;
    const float inv = nothing ? 0.f : 1.f / sum;
    u32x2* const at = (u32x2*)(p.out + (from + tok) * p.o_st + (int64_t)h * p.o_sh + d);
    *at = u32x2{Elem<T>::pack(o[0] * inv, o[1] * inv), Elem<T>::pack(o[2] * inv, o[3] * inv)};
    if (p.lse && d == 0)
      p.lse[(from + tok) * ((int64_t)p.kv_heads * p.group) + h] =
          nothing ? -__builtin_inff() : (top + __builtin_amdgcn_logf(sum)) * (1.f / kLog2e);
  }
}

// The prefill kernel's stages of LDS: arrays of their own, so that a load into one is no reason to wait
// before a read of another.
template <int D, int S>
__device__ __forceinline__ u32x4* prefill_stage() {
  __shared__ u32x4 stage[4 * 2 * D];  // four 16-token tiles of 32 D bytes
  return stage;
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t cache_rsrc(const uint8_t* base, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, bytes, 0x00020000);
}
// 16 bytes per lane straight into LDS, lane i's at lds + 16 i; out of range: zeros.
__device__ __forceinline__ void load_lds(__amdgpu_buffer_rsrc_t r, u32x4* lds, int lane_off, int off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, lane_off, off, 0, 0);
}
// Wait until at most N vector-memory loads of this wave are outstanding; they complete in order.
template <int N>
__device__ __forceinline__ void vmem_wait() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt((N & 0xF) | ((N >> 4) << 14) | (0x7 << 4) | (0xF << 8));
  __builtin_amdgcn_sched_barrier(0);
}

// ---------------------------------------------------------------------------------------------- host

struct Shape {
  int rows;             // of a work-group
  int32_t row_tiles;    // work-groups over the rows of a cached head
  int32_t splits;
  int32_t chunk;
};

int64_t workspace_bytes(const Shape& s, int32_t rows, int32_t kv_heads, int32_t d) {
  if (s.splits <= 1 || rows == 0) return 0;
  return BSG_KV_COUNTER_BYTES + (int64_t)rows * kv_heads * s.row_tiles * s.splits * s.rows * (d + 2) * 4;
}

int check_heads(const bsg_kv_cache* c, int32_t q_heads) {
  if (q_heads < 1 || q_heads % c->n_heads != 0)
    return fail(BSG_ERR_ARG, "q_heads=%d is no multiple of the cache's %d heads", q_heads, c->n_heads);
  return BSG_OK;
}

// What a call of either entry point is given.
struct AttnCall {
  const void* q;
  int64_t q_st, q_sh, tokens;
  int32_t q_heads;
  const bsg_kv_cache* cache;
  const int32_t* slots;
  int32_t rows;
  const int32_t* cu;
  int32_t max_new;
  float sm_scale;
  void* out;
  int64_t o_st, o_sh;
  float* lse;
  int dtype;
  void* ws;
  int64_t ws_bytes;
  int32_t cu_count;
};

int check_call(const AttnCall& c) {
  if (const int rc = check_kv_cache(c.cache)) return rc;
  if (const int rc = check_heads(c.cache, c.q_heads)) return rc;
  if (const int rc = check_kv_batch(c.tokens, c.rows, c.slots, c.cu, c.max_new, c.cache, c.dtype)) return rc;
  if (c.cu_count < 1) return fail(BSG_ERR_ARG, "cu_count=%d", c.cu_count);
  if (!(__builtin_fabsf(c.sm_scale * kLog2e) < __builtin_inff())) return fail(BSG_ERR_ARG, "sm_scale=%g", c.sm_scale);
  return BSG_OK;
}

// Of a call that has something to do.
int check_tensors(const AttnCall& c) {
  if (!c.q || !c.out) return fail(BSG_ERR_ARG, "null pointer (q=%p out=%p)", c.q, c.out);
  if (!is_aligned(c.q, 16) || ((c.q_st | c.q_sh) & 7) != 0)
    return fail(BSG_ERR_ALIGN, "q rows must be 16-byte aligned (strides %lld, %lld)", (long long)c.q_st, (long long)c.q_sh);
  if (!is_aligned(c.out, 8) || ((c.o_st | c.o_sh) & 3) != 0)
    return fail(BSG_ERR_ALIGN, "out rows must be 8-byte aligned (strides %lld, %lld)", (long long)c.o_st, (long long)c.o_sh);
  const int32_t group = c.q_heads / c.cache->n_heads;
  if ((int64_t)c.max_new * group > 0x7fffffff / 2) return fail(BSG_ERR_UNSUPPORTED, "%d tokens x %d heads", c.max_new, group);
  return BSG_OK;
}

// The kernels' parameters for a call that is cut as `s` says, once its workspace, of `need` bytes, has been looked at.
int call_params(const AttnCall& c, const Shape& s, int64_t need, AttnParams* p) {
  const bsg_kv_cache* const cache = c.cache;
  if (need > 0 && (!c.ws || c.ws_bytes < need))
    return fail(BSG_ERR_WORKSPACE, "workspace of %lld bytes, %lld needed", (long long)c.ws_bytes, (long long)need);
  if (need > 0 && !is_aligned(c.ws, 16)) return fail(BSG_ERR_ALIGN, "workspace must be 16-byte aligned");
  if ((int64_t)cache->n_heads * s.row_tiles > kLaunchGroups || c.rows > 65535 || s.row_tiles > 65535)
    return fail(BSG_ERR_UNSUPPORTED, "%d sequences of %d tokens", c.rows, c.max_new);
  p->q = (const uint16_t*)c.q;
  p->out = (uint16_t*)c.out;
  p->lse = c.lse;
  p->pages = (const uint8_t*)cache->pages;
  p->scales = cache->scales;
  p->table = cache->page_table;
  p->lengths = cache->lengths;
  p->slots = c.slots;
  p->cu = c.cu;
  p->parents = nullptr;
  p->counters = (uint32_t*)c.ws;
  p->part = need > 0 ? (float*)((uint8_t*)c.ws + BSG_KV_COUNTER_BYTES) : nullptr;
  p->q_st = c.q_st, p->q_sh = c.q_sh, p->o_st = c.o_st, p->o_sh = c.o_sh;
  p->table_stride = cache->table_stride;
  p->tokens = c.tokens;
  p->scale2 = c.sm_scale * kLog2e;
  p->num_pages = (int32_t)cache->num_pages;
  p->kv_heads = cache->n_heads;
  p->group = c.q_heads / cache->n_heads;
  p->num_slots = cache->num_slots;
  p->max_pages = cache->max_pages;
  p->page_shift = __builtin_ctz((unsigned)cache->page_size);
  p->max_new = c.max_new;
  p->row_tiles = s.row_tiles;
  p->splits = s.splits;
  p->chunk = s.chunk;
  return BSG_OK;
}

}  // namespace
