// kv_attention.hip — attention over the 8-bit paged cache (include/bsgserve.h).
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

#include <utility>

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

// A NaN among values that some rows do not see: the matrix unit would spread it to all rows (0 x
// NaN), so it goes to those that see it by a product of flags, and leaves the values.  v: four tiles of 16 channels
// of two 16-token tiles, t: the lane's first token, acc: their four accumulators of each 16 rows.
template <int RT>
__device__ __forceinline__ void nan_values(u32x4 v[2], int t, const int* sees, f32x4* acc, int stride) {
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    uint32_t f[4];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        f[2 * a + j] = Elem<_Float16>::pack(t + 16 * a + 2 * j < sees[i] ? 1.f : 0.f, t + 16 * a + 2 * j + 1 < sees[i] ? 1.f : 0.f);
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

// Sum of a tile's parts: `rows` rows of D numbers in each of `chunks` parts, every part times its
// factor, s_f[row * FL + 2 * part]; done(row, channel, sum) gets four numbers at a time.  Four rows' and
// two parts' loads are in flight for each thread.
template <int D, int FL, typename Done>
__device__ __forceinline__ void sum_parts(__amdgpu_buffer_rsrc_t r, int part_bytes, int row0, int rows, int chunks,
                                          const float* s_f, const Done& done) {
  constexpr int PER = D / 4, ITEMS = 4, PARTS = 2;
  for (int e0 = threadIdx.x; e0 < rows * PER; e0 += ITEMS * 256) {
    f32x4 o[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < chunks; s += PARTS) {
      f32x4 v[PARTS][ITEMS];
#pragma unroll
      for (int j = 0; j < PARTS; ++j)
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
          const int e = e0 + 256 * i;
          // an offset past the buffer loads zeros
          const int at = e < rows * PER && s + j < chunks ? (s + j) * part_bytes + (row0 * PER + e) * 16 : -1;
          v[j][i] = hand_load16(r, at);
        }
#pragma unroll
      for (int j = 0; j < PARTS; ++j)
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
          const int e = e0 + 256 * i;
          if (e < rows * PER && s + j < chunks) o[i] += v[j][i] * s_f[e / PER * FL + 2 * (s + j)];
        }
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int e = e0 + 256 * i;
      if (e < rows * PER) done(row0 + e / PER, e % PER * 4, o[i]);
    }
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
template <typename T, int D, int RT>
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
  const int all_see = first + rt * ROWS / p.group + 1;  // tokens that every row sees
  const int chunks = end <= p.chunk ? 1 : (end + p.chunk - 1) / p.chunk < p.splits ? (end + p.chunk - 1) / p.chunk : p.splits;
  if (split >= chunks) return;
  const int t_begin = split * p.chunk;
  const int t_end = split == chunks - 1 ? end : t_begin + p.chunk;

  // Q^T as the B operand: column = row of the tile, channels in the order the keys' tiles have them
  x8 qf[RT][2 * C];
  int sees[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int r = rt * ROWS + 16 * i + col;
    const int tok = r / p.group, h = r - tok * p.group;
    const bool on = 16 * i + col < rows;
    sees[i] = on ? first + tok + 1 : 0;
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
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            s[a][j] = s[a][j] * ks[a] + lv[a];
            if (partial && (!there[a] || t0 + 16 * a + 4 * g + j >= sees[i])) s[a][j] = -__builtin_inff();
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
          nan_values<RT>(v, t0 + 4 * g, sees, &acc[0][4 * c], DT);
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

// Many rows per cached head (prompts).  A work-group of four waves owns 128 rows, 32 of each wave, and walks the
// tokens they see 64 at a time; a step's keys and values (16 KiB) are brought once, straight into LDS in
// the bytes they have in memory, two steps ahead, and each wave converts what it reads (converted once
// for all four, LDS holds twice the bytes: 645 us against 584 for a prompt of 8192).  Rows do not cross waves,
// so nothing meets at the end but the parts of a split.  Work-groups of one cached head lie kv_heads
// apart, that is on the same XCD where the heads are a multiple of 8, and share its L2; one sequence
// follows the other (all of them side by side: 334 us against 267 for 8 prompts of 2048), its tiles with
// most tokens first.
//
// 3 prompts of up to 2000 tokens over up to 2800, 32 heads on 8 of 128, fp16: 152 us, 758 TFLOP/s; a prompt of
// 8192: 556 us, 989 TFLOP/s, 0.82 of a library product of 8192^3 (1210).  The conversions hide behind the
// MFMAs; the softmax between the two products, with two waves on a SIMD, and the step's barrier do not.
template <typename T, int D>
__global__ __launch_bounds__(256, 2) void bsg_kv_prefill_kernel(AttnParams p) {
  constexpr int C = D / 64, DT = D / 16, RT = 2, ROWS = 128, STEP = 64;
  typedef typename Elem<T>::x8 x8;
  constexpr int TILE = 2 * C * 64, LOADS = 2 * C;  // 16-byte pieces of a 16-token tile, keys then values; a wave's loads
  __shared__ uint32_t s_last;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, g = lane >> 4;
  const int head = blockIdx.x % p.kv_heads;
  const int split = blockIdx.y, row = blockIdx.z;

  const int slot = p.slots ? p.slots[row] : row;
  int64_t from = (int64_t)row * p.max_new, to = from + p.max_new;
  if (p.cu) from = p.cu[row], to = p.cu[row + 1];
  if (from < 0 || to > p.tokens || from >= to) return;
  const int count = (int)(to - from < p.max_new ? to - from : p.max_new);
  // a sequence's row tiles from its last one on, whatever the longest sequence of the call has
  const int rt = (count * p.group - 1) / ROWS - (int)(blockIdx.x / p.kv_heads);
  if (rt < 0) return;
  const int rows = count * p.group - rt * ROWS;
  const int used = rows < ROWS ? rows : ROWS;
  int len = slot >= 0 && slot < p.num_slots ? p.lengths[slot] : 0;
  const int most = p.max_pages << p.page_shift;
  len = len < 0 ? 0 : len > most ? most : len;
  const int first = len - (int)(to - from);
  const auto sees_until = [&](int r) {  // tokens that row r of the tile sees
    const int n = first + (rt * ROWS + r) / p.group + 1;
    return n < 0 ? 0 : n;
  };
  const int end = sees_until(used - 1);
  const int chunks = end <= p.chunk ? 1 : (end + p.chunk - 1) / p.chunk < p.splits ? (end + p.chunk - 1) / p.chunk : p.splits;
  if (split >= chunks) return;
  const int t_begin = split * p.chunk;
  const int t_end = split == chunks - 1 ? end : t_begin + p.chunk;
  // this wave's rows: 32 wave .. +31
  const int w_used = used - 32 * wave < 32 ? used - 32 * wave : 32;
  const int w_end = w_used > 0 ? sees_until(32 * wave + w_used - 1) : 0;  // what its last row sees
  const int w_all = w_used > 0 ? sees_until(32 * wave) : 0;               // what all of them see

  x8 qf[RT][2 * C];
  int sees[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int r = 32 * wave + 16 * i + col;
    const int rr = rt * ROWS + r, tok = rr / p.group, h = rr - tok * p.group;
    const bool on = r < used;
    sees[i] = on ? first + tok + 1 : 0;
#pragma unroll
    for (int c = 0; c < 2 * C; ++c) {
      u32x4 v = {0u, 0u, 0u, 0u};
      if (on)
        v = *(const u32x4*)(p.q + (from + tok) * p.q_st + (int64_t)(head * p.group + h) * p.q_sh + 64 * (c >> 1) +
                            16 * g + 8 * (c & 1));
      v ^= p.scale2 < 0.f ? 0x80008000u : 0u;  // so that the scores' scale is positive
      qf[i][c] = __builtin_bit_cast(x8, v);
    }
  }
  const float scale2 = __builtin_fabsf(p.scale2);

  const int32_t* const table = p.table + (int64_t)(slot < 0 || slot >= p.num_slots ? 0 : slot) * p.table_stride;
  const int64_t head_bytes = (int64_t)2 * D << p.page_shift;
  const int in_page = (1 << p.page_shift) - 1;
  // Lane j keeps where the j-th 16-token tile of 16 steps (1024 tokens) lies and its scales, from where
  // they come as scalars; the next 16 steps' are on their way while the last of these are at work.
  struct Tiles {
    int64_t at;  // bytes into the pages; below 0: not there
    float ks, lv, iv;
  } tiles = {-1, 0.f, 0.f, 0.f};
  int next_page = -1;
  int64_t next_at = -1;
  f32x2 next_scale = {0.f, 0.f};
  const auto load_pages = [&](int b0) {  // not looked at before load_scales
    const int t = b0 + 16 * lane;
    next_page = t < t_end ? table[t >> p.page_shift] : -1;
  };
  const auto load_scales = [&](int b0) {
    const bool there = next_page >= 0 && next_page < p.num_pages;
    const int64_t block = (int64_t)(there ? next_page : 0) * p.kv_heads + head;
    next_at = there ? block * head_bytes + (int64_t)(((b0 + 16 * lane) & in_page) * D) : -1;
    next_scale = *(const f32x2*)(p.scales + 2 * block);
  };
  const auto turn_pages = [&]() {
    const float vs = fmaxf(next_scale.y, 0x1p-100f);
    // a scale of 0 as the least one, so that -inf stays what it is
    tiles = Tiles{next_at, fmaxf(next_scale.x * scale2, 0x1p-126f), __builtin_amdgcn_logf(vs), __builtin_amdgcn_rcpf(vs)};
  };
  // The wave brings the tile `wave` of step n of the 16 (from 16 on: of the next 16); one that is not
  // there, or past the end, loads zeros, so that every step has the same number of loads to wait by.
  const auto issue = [&](auto stage, int n) {
    const int64_t from = n < 16 ? tiles.at : next_at;
    const int at = 4 * n + wave & 63;
    const int lo = __builtin_amdgcn_readlane((int)from, at), hi = __builtin_amdgcn_readlane((int)(from >> 32), at);
    const int64_t off = hi < 0 ? 0 : (int64_t)hi << 32 | (uint32_t)lo;
    const int half = (int)(head_bytes >> 1);
    const __amdgpu_buffer_rsrc_t r = cache_rsrc(p.pages + off, hi >= 0 ? half + 1024 * C : 0);
    u32x4* const to = prefill_stage<D, decltype(stage)::value>() + wave * TILE;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      load_lds(r, to + c * 64, lane * 16, c * 1024);
      load_lds(r, to + (C + c) * 64, lane * 16, c * 1024 + half);
    }
  };

  f32x4 acc[RT][DT];
  float base[RT], l[RT];  // -inf: no token seen
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    base[i] = -__builtin_inff(), l[i] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[i][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  bool started = false;  // every row has a base, and one that is not far
  const auto take = [&](auto stage, int t0) {
    const u32x4* const kv = prefill_stage<D, decltype(stage)::value>() + lane;
    const int first_tile = (t0 - t_begin) / 16 & 63;
    f32x4 s[RT][4];
    float ks[4], lv[4], iv[4];
    bool there[4], all_there = true;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      there[a] = __builtin_amdgcn_readlane((int)(tiles.at >> 32), first_tile + a) >= 0;
      ks[a] = as_float(__builtin_amdgcn_readlane(__builtin_bit_cast(int, tiles.ks), first_tile + a));
      lv[a] = as_float(__builtin_amdgcn_readlane(__builtin_bit_cast(int, tiles.lv), first_tile + a));
      iv[a] = as_float(__builtin_amdgcn_readlane(__builtin_bit_cast(int, tiles.iv), first_tile + a));
      all_there = all_there && there[a];
#pragma unroll
      for (int i = 0; i < RT; ++i) s[i][a] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const u32x4 k = kv[a * TILE + c * 64];
        const x8 k0 = widen<T>(k.x, k.y), k1 = widen<T>(k.z, k.w);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          s[i][a] = Elem<T>::mfma(k0, qf[i][2 * c], s[i][a]);
          s[i][a] = Elem<T>::mfma(k1, qf[i][2 * c + 1], s[i][a]);
        }
      }
    }
    const bool partial = t0 + STEP > w_all || !all_there;
    if (partial) {
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const int t = there[a] ? t0 + 16 * a + 4 * g : 0x7ffffff0;
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (t + j >= sees[i]) s[i][a][j] = -__builtin_inff();
      }
    }
    // Weights against the base so far; only where four of them together outgrow fp16 (or a row has no
    // base yet, or a far one) is a new one looked for.  The sums are wanted anyway: asking each weight took 590 us
    // instead of 566 for a prompt of 8192.  Against a new base the score is rounded first, so that the maximum's
    // weight is 2^13 or 1 however far it is; otherwise both come in one step.
    f16x8 pf[RT][2];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      float e[4][4], sum[4], top = 0.f;
      const auto weigh = [&](auto exactly) {
        const float from = base[i] == -__builtin_inff() ? 0.f : base[i];
        top = 0.f;
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const float off = lv[a] - from;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            e[a][j] = __builtin_amdgcn_exp2f(decltype(exactly)::value ? __builtin_fmaf(s[i][a][j], ks[a], lv[a]) - from
                                                                      : __builtin_fmaf(s[i][a][j], ks[a], off));
          sum[a] = (e[a][0] + e[a][1]) + (e[a][2] + e[a][3]);
          top = fmaxf(top, sum[a]);
        }
      };
      weigh(std::false_type{});
      if (!started || __any(top > kMostWeight)) {
        float mx = -__builtin_inff();
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const float t = fmaxf(fmaxf(s[i][a][0], s[i][a][1]), fmaxf(s[i][a][2], s[i][a][3]));
          mx = fmaxf(mx, __builtin_fmaf(t, ks[a], lv[a]));
        }
        mx = column_max(mx);
        const float next = fmaxf(base[i], base_of(mx));
        const float alpha = next == base[i] ? 1.f : __builtin_amdgcn_exp2f(base[i] - next);
        l[i] *= alpha;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[i][d] *= alpha;
        base[i] = next;
        started = false;
        weigh(std::true_type{});
      }
      uint32_t w[8];
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        l[i] = __builtin_fmaf(sum[a], iv[a], l[i]);
        w[2 * a] = Elem<_Float16>::pack(e[a][0], e[a][1]), w[2 * a + 1] = Elem<_Float16>::pack(e[a][2], e[a][3]);
      }
      pf[i][0] = __builtin_bit_cast(f16x8, u32x4{w[0], w[1], w[2], w[3]});
      pf[i][1] = __builtin_bit_cast(f16x8, u32x4{w[4], w[5], w[6], w[7]});
    }
    if (!started)
      started = !partial && !__any(!(__builtin_fabsf(base[0]) < kFarScore) || !(__builtin_fabsf(base[1]) < kFarScore));
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        u32x4 v[2] = {kv[2 * b * TILE + (C + c) * 64], kv[(2 * b + 1) * TILE + (C + c) * 64]};
        if (partial) {
          uint32_t nan = 0;
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            v[a] &= there[2 * b + a] ? byte_mask(t_end - (t0 + 32 * b + 16 * a + 4 * g)) : 0u;
            nan |= nan_bytes(v[a].x) | nan_bytes(v[a].y) | nan_bytes(v[a].z) | nan_bytes(v[a].w);
          }
          if (__any(nan != 0)) nan_values<RT>(v, t0 + 32 * b + 4 * g, sees, &acc[0][4 * c], DT);
        }
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const f16x8 x = widen<_Float16>(v[0][d], v[1][d]);
#pragma unroll
          for (int i = 0; i < RT; ++i) acc[i][4 * c + d] = Elem<_Float16>::mfma(x, pf[i][b], acc[i][4 * c + d]);
        }
      }
    }
  };

  if (t_begin < t_end) {
    load_pages(t_begin);
    load_scales(t_begin);
    tiles.at = next_at;
    issue(std::integral_constant<int, 0>{}, 0);
    issue(std::integral_constant<int, 1>{}, 1);
    turn_pages();
    int n = 0;
    for (int t0 = t_begin; t0 < t_end; t0 += 3 * STEP)
      [&]<int... I>(std::integer_sequence<int, I...>) {
        (..., [&](auto stage) {
          constexpr int S = decltype(stage)::value;
          const int t = t0 + S * STEP;
          // this step's pieces have arrived for every wave, and every wave has read the step's before
          vmem_wait<LOADS>();
          __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
          asm volatile("" ::: "memory");
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
          __builtin_amdgcn_sched_barrier(0);
          if (n == 8) load_pages(t + 8 * STEP);
          if (n == 11) load_scales(t + 5 * STEP);
          issue(std::integral_constant<int, (S + 2) % 3>{}, n + 2);
          __builtin_amdgcn_sched_barrier(0);
          if (t < w_end && t < t_end) take(stage, t);
          if (++n == 16) n = 0, turn_pages();
        }(std::integral_constant<int, I>{}));
      }(std::make_integer_sequence<int, 3>{});
    vmem_wait<0>();  // nothing is on its way into LDS any more
  }
#pragma unroll
  for (int i = 0; i < RT; ++i) l[i] = column_sum(l[i]);

  const int64_t heads = (int64_t)p.kv_heads * p.group;
  const auto finish = [&](int r, int d, f32x4 o, float top, float sum) {
    const int rr = rt * ROWS + r, tok = rr / p.group, h = head * p.group + rr - tok * p.group;
    const bool nothing = sum == 0.f;
    const float inv = nothing ? 0.f : 1.f / sum;
    u32x2* const at = (u32x2*)(p.out + (from + tok) * p.o_st + (int64_t)h * p.o_sh + d);
    *at = u32x2{Elem<T>::pack(o[0] * inv, o[1] * inv), Elem<T>::pack(o[2] * inv, o[3] * inv)};
    if (p.lse && d == 0)
      p.lse[(from + tok) * heads + h] =
          nothing ? -__builtin_inff() : (top + __builtin_amdgcn_logf(sum)) * (1.f / kLog2e);
  };
  if (chunks == 1) {
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int r = 32 * wave + 16 * i + col;
      if (r < used) {
#pragma unroll
        for (int d = 0; d < DT; ++d) finish(r, 16 * d + 4 * g, acc[i][d], base[i], l[i]);
      }
    }
    return;
  }

  const int64_t tile = ((int64_t)row * p.kv_heads + head) * p.row_tiles + rt;
  constexpr int PART = ROWS * (D + 2);
  const float* const parts = p.part + tile * p.splits * PART;
  float* const part = p.part + (tile * p.splits + split) * PART;
  const __amdgpu_buffer_rsrc_t mine_rsrc = hand_buffer(part, PART * 4);
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int r = 32 * wave + 16 * i + col;
    if (r < used) {
#pragma unroll
      for (int d = 0; d < DT; ++d) hand_store16(mine_rsrc, (r * D + 16 * d + 4 * g) * 4, acc[i][d]);
      if (g == 0) hand_store((uint64_t*)(part + ROWS * D) + r, __builtin_bit_cast(uint64_t, f32x2{base[i], l[i]}));
    }
  }
  hand_publish();
  __syncthreads();
  if (threadIdx.x == 0) s_last = hand_arrive(p.counters + tile) == (uint32_t)(chunks - 1);
  __syncthreads();
  if (!s_last) return;
  if (threadIdx.x == 0) hand_reset(p.counters + tile);
  // [row][part] factors and, in the row's first pair, the base and the sum
  float* const s_f = (float*)prefill_stage<D, 0>();
  constexpr int FL = 2 * kMaxSplits;
  constexpr int BLOCK = 4 * TILE * 16 / (FL * 4);  // rows whose factors fit a stage at once
  for (int r0 = 0; r0 < used; r0 += BLOCK) {
    const int n = used - r0 < BLOCK ? used - r0 : BLOCK;
    __syncthreads();
    for (int e = threadIdx.x; e < n * chunks; e += 256) {
      const int r = e / chunks, s = e - r * chunks;
      const f32x2 v = __builtin_bit_cast(f32x2, hand_load((const uint64_t*)(parts + s * PART + ROWS * D) + r0 + r));
      s_f[r * FL + 2 * s] = v.x, s_f[r * FL + 2 * s + 1] = v.y;
    }
    __syncthreads();
    if ((int)threadIdx.x < n) {
      float* const f = s_f + threadIdx.x * FL;
      float top = -__builtin_inff(), sum = 0.f;
      for (int s = 0; s < chunks; ++s) top = fmaxf(top, f[2 * s]);
      for (int s = 0; s < chunks; ++s) {
        f[2 * s] = f[2 * s] == top ? 1.f : __builtin_amdgcn_exp2f(f[2 * s] - top);
        sum += f[2 * s] * f[2 * s + 1];
      }
      f[1] = top, f[3] = sum;  // at least two parts
    }
    __syncthreads();
    sum_parts<D, FL>(hand_buffer(parts, chunks * PART * 4), PART * 4, r0, n, chunks, s_f,
                     [&](int r, int d, f32x4 o) { finish(r, d, o, s_f[(r - r0) * FL + 1], s_f[(r - r0) * FL + 3]); });
  }
}

struct Shape {
  int rows;             // of a work-group
  int32_t row_tiles;    // work-groups over the rows of a cached head
  int32_t splits;
  int32_t chunk;
};

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

int64_t workspace_bytes(const Shape& s, int32_t rows, int32_t kv_heads, int32_t d) {
  if (s.splits <= 1 || rows == 0) return 0;
  return BSG_KV_COUNTER_BYTES + (int64_t)rows * kv_heads * s.row_tiles * s.splits * s.rows * (d + 2) * 4;
}

template <typename T, int D>
void launch(const AttnParams& p, const Shape& s, dim3 grid, hipStream_t st) {
  switch (s.rows) {
    case 16: hipLaunchKernelGGL((bsg_kv_attention_kernel<T, D, 1>), grid, dim3(256), 0, st, p); break;
    case 32: hipLaunchKernelGGL((bsg_kv_attention_kernel<T, D, 2>), grid, dim3(256), 0, st, p); break;
    default: hipLaunchKernelGGL((bsg_kv_prefill_kernel<T, D>), grid, dim3(256), 0, st, p); break;
  }
}

int check_heads(const bsg_kv_cache* c, int32_t q_heads) {
  if (q_heads < 1 || q_heads % c->n_heads != 0)
    return fail(BSG_ERR_ARG, "q_heads=%d is no multiple of the cache's %d heads", q_heads, c->n_heads);
  return BSG_OK;
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
  if (const int rc = check_kv_cache(cache)) return rc;
  if (const int rc = check_heads(cache, q_heads)) return rc;
  if (const int rc = check_kv_batch(tokens, rows, slots, cu, max_new, cache, dtype)) return rc;
  if (cu_count < 1) return fail(BSG_ERR_ARG, "cu_count=%d", cu_count);
  if (!(__builtin_fabsf(sm_scale * kLog2e) < __builtin_inff())) return fail(BSG_ERR_ARG, "sm_scale=%g", sm_scale);
  if (tokens == 0 || rows == 0 || max_new == 0) return BSG_OK;
  if (!q || !out) return fail(BSG_ERR_ARG, "null pointer (q=%p out=%p)", q, out);
  if (!is_aligned(q, 16) || ((q_stride_t | q_stride_h) & 7) != 0)
    return fail(BSG_ERR_ALIGN, "q rows must be 16-byte aligned (strides %lld, %lld)", (long long)q_stride_t,
                (long long)q_stride_h);
  if (!is_aligned(out, 8) || ((o_stride_t | o_stride_h) & 3) != 0)
    return fail(BSG_ERR_ALIGN, "out rows must be 8-byte aligned (strides %lld, %lld)", (long long)o_stride_t,
                (long long)o_stride_h);
  const int64_t most = (int64_t)cache->max_pages * cache->page_size;
  if (max_len <= 0 || max_len > most) max_len = most;
  const int32_t group = q_heads / cache->n_heads;
  if ((int64_t)max_new * group > 0x7fffffff / 2) return fail(BSG_ERR_UNSUPPORTED, "%d tokens x %d heads", max_new, group);
  const Shape s = shape_of(rows, cache->n_heads, group, max_new, max_len, cu_count);
  const int64_t need = workspace_bytes(s, rows, cache->n_heads, cache->head_dim);
  if (need > 0 && (!ws || ws_bytes < need))
    return fail(BSG_ERR_WORKSPACE, "workspace of %lld bytes, %lld needed", (long long)ws_bytes, (long long)need);
  if (need > 0 && !is_aligned(ws, 16)) return fail(BSG_ERR_ALIGN, "workspace must be 16-byte aligned");
  const int64_t gx = (int64_t)cache->n_heads * s.row_tiles;
  if (gx > kLaunchGroups || rows > 65535 || s.row_tiles > 65535)
    return fail(BSG_ERR_UNSUPPORTED, "%d sequences of %d tokens", rows, max_new);
  AttnParams p;
  p.q = (const uint16_t*)q;
  p.out = (uint16_t*)out;
  p.lse = lse;
  p.pages = (const uint8_t*)cache->pages;
  p.scales = cache->scales;
  p.table = cache->page_table;
  p.lengths = cache->lengths;
  p.slots = slots;
  p.cu = cu;
  p.counters = (uint32_t*)ws;
  p.part = need > 0 ? (float*)((uint8_t*)ws + BSG_KV_COUNTER_BYTES) : nullptr;
  p.q_st = q_stride_t, p.q_sh = q_stride_h, p.o_st = o_stride_t, p.o_sh = o_stride_h;
  p.table_stride = cache->table_stride;
  p.tokens = tokens;
  p.scale2 = sm_scale * kLog2e;
  p.num_pages = (int32_t)cache->num_pages;
  p.kv_heads = cache->n_heads;
  p.group = group;
  p.num_slots = cache->num_slots;
  p.max_pages = cache->max_pages;
  p.page_shift = __builtin_ctz((unsigned)cache->page_size);
  p.max_new = max_new;
  p.row_tiles = s.row_tiles;
  p.splits = s.splits;
  p.chunk = s.chunk;
  const dim3 grid((unsigned)gx, (unsigned)s.splits, (unsigned)rows);
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == BSG_F16)
    cache->head_dim == 64 ? launch<_Float16, 64>(p, s, grid, st) : launch<_Float16, 128>(p, s, grid, st);
  else
    cache->head_dim == 64 ? launch<__bf16, 64>(p, s, grid, st) : launch<__bf16, 128>(p, s, grid, st);
  return launch_status("bsg_kv_attention");
}
