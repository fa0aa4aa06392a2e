// logprobs.hip — log probabilities of given tokens, entropies and the likeliest alternatives of rows of
// logits, in one pass over them (include/bsgserve.h).
//
// With a reference M near the row's maximum, d = (x - M) log2(e), l = sum 2^d and t = sum 2^d d:
//   logprob = ln 2 (d_token - log2 l),  entropy = ln 2 (log2 l - t / l).
// Any M gives the same, so a wave keeps its first tile's maximum until a logit is kSlack above it: close to the
// row's, since the entropy is what log2 l and t / l differ by, and they are as large as the maximum lies above M.
// Where |M| is below kFar what log2(e) M is rounded to cancels: d is one fused multiply-add.  From there on (masks are
// logits too, and a wave may have nothing else) the rounding alone would be octaves, so x - M comes first.
//
// The alternatives are found beside it.  A logit's key is its order among fp32 numbers (upper half) and
// its id's complement (lower half), so that keys are distinct and (logit desc, id asc) is key desc.
// The unit of work is a wave: it keeps the 64 best keys of its slice sorted, one per lane, and
// compares what it reads with the k-th of them; what passes waits in LDS and is merged 64 at a time by
// bitonic networks over DPP moves.  Before the first tile there is nothing to compare with: the k-th
// largest of the lanes' own maxima is a bound that at least k logits reach.  Waves of a row meet in
// LDS, two lists at a time; no barrier before that.
//
// 4000 x 32000 bf16 (256 MB): 49 us without alternatives (5.3 TB/s, past the rate of a copy), 52 with one, 63 with
// 8, 87 with 50 (fp16): what is left of the sorts, of which every wave runs two.  64 x 32000 fp16: 8.3 us without,
// 13.0 with 8, bound by the chain of loads, sort, insertions and the three meetings of eight waves.

#include "serve.hpp"

using namespace bsgk;

namespace {

constexpr int kVectors = 4;     // 16-byte vectors of a lane and tile
constexpr int kAhead = 1;       // tiles in flight beside the one at work
constexpr int kWaves = 4;       // of a work-group of several rows, or of a row's split
constexpr int kMostWaves = 8;   // of a work-group that has a row to itself
constexpr int kInsert = 16;     // keys up to which inserting one by one is quicker than a sort
constexpr int kSplitTiles = 2;  // tiles of a wave that a split of a long row leaves
constexpr int kMaxSplits = 32;  // of a row
constexpr int kMaxK = BSG_LOGPROBS_MAX_K;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kSlack = 2.f;  // weights stay below 2^3
constexpr float kFar = 0x1p20f;  // references from here on: log2(e) M is off by 2^-4 octaves and more, differences before products
constexpr float kHuge = 1e38f;  // logits from here on: log2(e) (x - M) may overflow where x - M does not
constexpr float kLow = -1e30f;  // below it (masks) 2^d d is not formed from d as it is
constexpr float kFloor = -1e4f;  // exponents below it weigh nothing; keeps 0 x -inf out of t

struct ScoreParams {
  const void* x;
  const int32_t* tokens;
  float* logprob;
  float* entropy;
  int32_t* top_ids;
  float* top_logprobs;
  uint32_t* counters;  // [rows]
  uint64_t* keys;      // [rows][splits][k]
  float* sums;         // [rows][splits][4]
  int64_t stride, vocab, split_vectors;
  int32_t rows, k, splits, log_waves;  // waves of a row and split: 1 << log_waves
};

template <typename T>
struct Logit;
template <>
struct Logit<_Float16> {
  static constexpr int N = 8;
  static constexpr uint32_t kMinusInf = 0xfc00u;
  static __device__ __forceinline__ float at(const u32x4& v, int i) {
    return i & 1 ? high_half<_Float16>(v[i >> 1]) : low_half<_Float16>(v[i >> 1]);
  }
};
template <>
struct Logit<__bf16> {
  static constexpr int N = 8;
  static constexpr uint32_t kMinusInf = 0xff80u;
  static __device__ __forceinline__ float at(const u32x4& v, int i) {
    return i & 1 ? high_half<__bf16>(v[i >> 1]) : low_half<__bf16>(v[i >> 1]);
  }
};
template <>
struct Logit<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float at(const u32x4& v, int i) { return as_float(v[i]); }
};

// fp32 numbers as unsigned ones in the same order: -0 equals +0, every NaN is the largest; no
// number gives 0.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
  const uint32_t o = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
  return x != x ? 0xffffffffu : o;
}
__device__ __forceinline__ float from_order(uint32_t o) {
  if (o == 0xffffffffu) return __builtin_nanf("");
  return __builtin_bit_cast(float, o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ uint64_t key_of(uint32_t order, uint32_t id) { return (uint64_t)order << 32 | (uint32_t)~id; }

// One step of a bitonic network of one value per lane: blocks of N sorted, every second the other
// way round, the last (N = 64) largest first.
template <int N, int X, typename V>
__device__ __forceinline__ V exchange(V v) {
  const V o = lane_xor<X>(v);
  const bool larger = ((threadIdx.x & X) == 0) == (N == 64 || (threadIdx.x & N) == 0);
  return (v > o) == larger ? v : o;
}
template <int N, int X, typename V>
__device__ __forceinline__ V merge_steps(V v) {
  v = exchange<N, X>(v);
  if constexpr (X > 1) v = merge_steps<N, X / 2>(v);
  return v;
}
template <int N, typename V>
__device__ __forceinline__ V sort_steps(V v) {
  if constexpr (N > 2) v = sort_steps<N / 2>(v);
  return merge_steps<N, N / 2>(v);
}
// Sorted, the largest in lane 0, or in lane 63.
template <typename V>
__device__ __forceinline__ V sorted_down(V v) {
  return sort_steps<64>(v);
}
template <typename V>
__device__ __forceinline__ V sorted_up(V v) {
  return (V)~sort_steps<64>((V)~v);
}
// The 64 largest of two lists, the first largest first, the second largest last; largest first.
__device__ __forceinline__ uint64_t merged(uint64_t down, uint64_t up) {
  return merge_steps<64, 32>(down > up ? down : up);
}

struct Sums {
  float m, l, t;  // l and t against the reference m, which a wave's lanes share while they read; -inf: nothing yet
};
__device__ __forceinline__ bool is_far(float m) { return !(__builtin_fabsf(m) < kFar); }
// (x - m) log2(e)
__device__ __forceinline__ float octaves(float x, float m) {
  return is_far(m) ? (x - m) * kLog2e : __builtin_fmaf(x, kLog2e, -(m * kLog2e));
}
// Octaves from reference m to a, each as sums against it have it: rounded after the product where it is not far.
__device__ __forceinline__ float between(float a, float m) {
#pragma clang fp contract(off)
  const float pa = a * kLog2e, pm = m * kLog2e;
  if (is_far(m)) return is_far(a) ? (a - m) * kLog2e : __builtin_fmaf(-m, kLog2e, pa);
  return is_far(a) ? __builtin_fmaf(a, kLog2e, -pm) : pa - pm;
}
__device__ __forceinline__ Sums join(Sums a, Sums b) {
#pragma clang fp contract(off)
  const float m = fmaxf(a.m, b.m);
  if (m == -__builtin_inff()) return Sums{m, a.l + b.l, a.t + b.t};
  const float da = fmaxf(between(a.m, m), kFloor), db = fmaxf(between(b.m, m), kFloor);
  const float fa = __builtin_amdgcn_exp2f(da), fb = __builtin_amdgcn_exp2f(db);
  return Sums{m, a.l * fa + b.l * fb, fa * (a.t + a.l * da) + fb * (b.t + b.l * db)};
}
template <int X>
__device__ __forceinline__ float max_lanes(float v) {
  v = fmaxf(v, lane_xor<X>(v));
  if constexpr (X < 32) v = max_lanes<2 * X>(v);
  return v;
}
template <int X>
__device__ __forceinline__ float add_lanes(float v) {
  v += lane_xor<X>(v);
  if constexpr (X < 32) v = add_lanes<2 * X>(v);
  return v;
}
template <int X>
__device__ __forceinline__ Sums join_lanes(Sums s) {
  s = join(s, Sums{lane_xor<X>(s.m), lane_xor<X>(s.l), lane_xor<X>(s.t)});
  if constexpr (X < 32) s = join_lanes<2 * X>(s);
  return s;
}

// What a wave keeps of its slice.
struct Best {
  uint64_t list;    // lane i: the i-th best key so far (0: none)
  uint64_t* wait;   // 128 keys of LDS, and a tile behind them
  int waiting;      // of them in use, below 64 between calls
  uint32_t bar;     // order that at least k logits of the slice so far reach; 0: fewer than k so far

  // What waits goes into the list: a few keys one after the other, many by a sort.
  __device__ __forceinline__ void settle(int k) {
    const int lane = threadIdx.x & 63;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const uint64_t v = lane < waiting ? wait[lane] : 0;
    const uint64_t rest = wait[64 + lane];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (waiting <= kInsert) {
      for (int i = 0; i < waiting; ++i) {
        const uint64_t key = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), i) << 32 |
                             (uint32_t)__builtin_amdgcn_readlane((int)v, i);
        const int at = __popcll(__ballot(list > key));
        const uint64_t above = (uint64_t)(uint32_t)__builtin_amdgcn_mov_dpp((int)(list >> 32), 0x138, 0xf, 0xf, true) << 32 |
                               (uint32_t)__builtin_amdgcn_mov_dpp((int)list, 0x138, 0xf, 0xf, true);  // wave_shr:1
        list = lane < at ? list : lane == at ? key : above;
      }
      waiting = 0;
    } else {
      if (waiting > 64 && lane < waiting - 64) wait[lane] = rest;
      waiting = waiting > 64 ? waiting - 64 : 0;
      list = merged(list, sorted_up(v));
    }
    const uint32_t kth = (uint32_t)__builtin_amdgcn_readlane((int)(list >> 32), k - 1);
    bar = bar > kth ? bar : kth;
  }
  __device__ __forceinline__ void add(bool take, uint64_t key) {
    const uint64_t who = __ballot(take);
    const int at = waiting + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0u));
    if (take) wait[at] = key;
    waiting += __popcll(who);
  }
};

// Vectors v0 + 64 i + lane of a row, of those before v_end.  A vector is an aligned 16-byte granule with
// at least one logit of the row in it.
__device__ __forceinline__ void load_tile(u32x4 raw[kVectors], const u32x4* row, int64_t v0, int64_t v_end) {
  const int lane = threadIdx.x & 63;
  const u32x4* const from = row + v0;
  const int64_t left = v_end - v0 - lane;
#pragma unroll
  for (int i = 0; i < kVectors; ++i)
    if (64 * i < left) raw[i] = __builtin_nontemporal_load(from + 64 * i + lane);
}

// What of a tile is no logit of the row (id0: the first lane's first id) becomes -inf; the bits of what is.
template <typename T>
__device__ __forceinline__ uint32_t clip_tile(u32x4 raw[kVectors], int64_t id0, int64_t v_left, int64_t vocab) {
  constexpr int N = Logit<T>::N;
  const int lane = threadIdx.x & 63;
  uint32_t there = 0;
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    const int64_t e = id0 + (int64_t)(64 * i + lane) * N;
    const int lo = e < 0 ? (int)-e : 0, hi = vocab - e < N ? (int)(vocab - e < 0 ? 0 : vocab - e) : N;
    const uint32_t bits = 64 * i + lane < v_left && lo < hi ? ((1u << hi) - 1u) & ~((1u << lo) - 1u) : 0u;
    there |= bits << (i * N);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if constexpr (sizeof(T) == 4) {
        if (!(bits >> w & 1u)) raw[i][w] = 0xff800000u;
      } else {
        const uint32_t keep = (bits >> (2 * w) & 1u ? 0xffffu : 0u) | (bits >> (2 * w + 1) & 1u ? 0xffff0000u : 0u);
        constexpr uint32_t inf = Logit<T>::kMinusInf;
        raw[i][w] = (raw[i][w] & keep) | ((inf | inf << 16) & ~keep);
      }
    }
  }
  return there;
}

// A tile into the sums and the alternatives; there: a bit for each of the lane's logits that is one of
// the row (the others are -inf); used: the vectors that any lane has.
template <typename T>
__device__ __forceinline__ void take_tile(const u32x4 raw[kVectors], uint32_t there, int used, int64_t id0, int k, bool first, Sums& sum,
                                          Best& best) {
  typedef Logit<T> L;
  constexpr int N = L::N;
  const int lane = threadIdx.x & 63;
  float top = -__builtin_inff(), low = __builtin_inff(), tops[kVectors];
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    tops[i] = -__builtin_inff();
    if (i < used) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float v = L::at(raw[i], j);
        tops[i] = fmaxf(tops[i], v);
        low = fminf(low, v);
      }
    }
    top = fmaxf(top, tops[i]);
  }
  float l = 0.f, t = 0.f;
  if (!__any(top > sum.m + kSlack || low < kLow || is_far(sum.m))) {
    const float base = sum.m * kLog2e;
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
      if (i < used) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float d = __builtin_fmaf(L::at(raw[i], j), kLog2e, -base);
          const float e = __builtin_amdgcn_exp2f(d);
          l += e;
          t = __builtin_fmaf(e, d, t);
        }
      }
  } else {  // a new reference, or numbers that need care
    const float high = max_lanes<1>(top);
    if (high > sum.m) sum = join(sum, Sums{high, 0.f, 0.f});
    const float m = sum.m == -__builtin_inff() ? 0.f : sum.m;
    // (x - m) log2(e), with the difference first or last
    const bool far = is_far(m);
    const float c = far ? 0.f : -(m * kLog2e), u = far ? m : 0.f;
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
      if (i < used) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float d = __builtin_fmaf(L::at(raw[i], j) - u, kLog2e, c);
          const float e = __builtin_amdgcn_exp2f(d);
          l += e;
          t = __builtin_fmaf(e, fmaxf(d, kFloor), t);
        }
      }
  }
  sum.l += l, sum.t += t;
  if (k == 0) return;

  if (first) {
    uint32_t mine = there != 0 ? order_of(top) : 0;
    if (l != l) {  // a NaN or +inf among them
#pragma unroll
      for (int i = 0; i < kVectors; ++i)
        if (i < used) {
#pragma unroll
          for (int j = 0; j < N; ++j)
            if (L::at(raw[i], j) != L::at(raw[i], j)) mine = 0xffffffffu;
        }
    }
    // what equals the bar enters too: of the k at or above it the ids are not known
    const uint32_t kth = (uint32_t)__builtin_amdgcn_readlane((int)sorted_down(mine), k - 1);
    best.bar = kth < 2 ? 0 : kth - (kth == 0x80000000u ? 2 : 1);  // below +0 comes -0, its equal
  }
  // The bar as a number; what is above it enters, and a NaN.  No number is above a bar of +inf, every
  // one above a bar of NaN, which stands for fewer than k keys so far.
  const float bar = best.bar == 0 ? __builtin_nanf("") : best.bar >= 0xff800000u ? __builtin_inff() : from_order(best.bar);
  const bool nan = l != l;
  if (!__any(!(top <= bar) || nan)) return;

  // Few enter; each lane takes its own one at a time, by position, from a copy of the tile in LDS.
  uint32_t mask = 0;
  u32x4* const copy = (u32x4*)(best.wait + 128);
#pragma unroll
  for (int i = 0; i < kVectors; ++i)
    if (i < used && __any(!(tops[i] <= bar) || nan)) {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (!(L::at(raw[i], j) <= bar)) mask |= 1u << (i * N + j);
      copy[64 * i + lane] = raw[i];
    }
  mask &= there;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  for (bool more = __any(mask != 0); more;) {
    const int bit = mask != 0 ? __builtin_ctz(mask) : 0;
    const int e = (64 * (bit / N) + lane) * N + bit % N;
    best.add(mask != 0, key_of(order_of((float)((const T*)copy)[e]), (uint32_t)(id0 + e)));
    mask &= mask - 1;
    more = __any(mask != 0);
    while (best.waiting >= 64 || (!more && best.waiting > 0)) best.settle(k);
  }
}

template <typename T, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void bsg_token_logprobs_kernel(ScoreParams p) {
  typedef Logit<T> L;
  constexpr int N = L::N;
  __shared__ alignas(16) uint64_t s_wait[WAVES][128 + 2 * 64 * kVectors];
  __shared__ Sums s_sum[WAVES];
  __shared__ uint32_t s_last;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int W = 1 << p.log_waves, part = wave & (W - 1);
  const int64_t row = (int64_t)blockIdx.y * (WAVES >> p.log_waves) + (wave >> p.log_waves);
  const bool real = row < p.rows;
  const T* const x = (const T*)p.x + (real ? row : 0) * p.stride;
  const int k = p.k;
  const int32_t token = real ? p.tokens[row] : -1;

  // 16-byte vectors from the granule in which the row begins: its element i is at i + skip
  const int skip = (int)(((uintptr_t)x & 15u) / sizeof(T));
  const int64_t vectors = real ? (p.vocab + skip + N - 1) / N : 0;
  const int64_t s_begin = (int64_t)blockIdx.x * p.split_vectors;
  const int64_t s_end = s_begin + p.split_vectors < vectors ? s_begin + p.split_vectors : vectors;
  const int64_t per = (p.split_vectors + W - 1) >> p.log_waves;
  const int64_t v_begin = s_begin + part * per;
  const int64_t v_end = v_begin + per < s_end ? v_begin + per : s_end;

  Sums sum = {-__builtin_inff(), 0.f, 0.f};
  Best best = {0, s_wait[wave], 0, 0};
  constexpr int STEP = 64 * kVectors;
  const u32x4* const granules = (const u32x4*)(x - skip);
  u32x4 next[kAhead][kVectors];
#pragma unroll
  for (int a = 0; a < kAhead; ++a) load_tile(next[a], granules, v_begin + a * STEP, v_end);
  const bool token_there = token >= 0 && token < p.vocab;
  const float token_logit = token_there ? (float)x[token] : __builtin_nanf("");
  for (int64_t v0 = v_begin; v0 < v_end; v0 += STEP) {
    u32x4 raw[kVectors];
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      raw[i] = next[0][i];
#pragma unroll
      for (int a = 1; a < kAhead; ++a) next[a - 1][i] = next[a][i];
    }
    load_tile(next[kAhead - 1], granules, v0 + kAhead * STEP, v_end);
    const int64_t id0 = v0 * N - skip;
    uint32_t there = 0xffffffffu;
    if (id0 < 0 || v0 + STEP > v_end || id0 + STEP * N > p.vocab) there = clip_tile<T>(raw, id0, v_end - v0, p.vocab);
    const int used = v0 + STEP <= v_end ? kVectors : (int)((v_end - v0 + 63) >> 6);
    take_tile<T>(raw, there, used, id0, k, v0 == v_begin, sum, best);
  }
  sum.l = add_lanes<1>(sum.l), sum.t = add_lanes<1>(sum.t);

  // the waves of a row, two at a time; the lists go through the waves' own LDS
  const auto meet = [&]() {
    for (int step = 1; step < W; step <<= 1) {
      if (part & step) {
        s_wait[wave][lane] = best.list;
        if (lane == 0) s_sum[wave] = sum;
      }
      __syncthreads();
      if ((part & (2 * step - 1)) == 0) {
        if (k > 0) best.list = merged(best.list, s_wait[wave + step][63 - lane]);
        sum = join(sum, s_sum[wave + step]);
      }
    }
  };
  meet();

  if (p.splits > 1) {
    const int64_t at = row * p.splits + blockIdx.x;
    if (part == 0 && real) {
      if (lane < k) hand_store(p.keys + at * k + lane, best.list);
      if (lane == 0) hand_store16(hand_buffer(p.sums + at * 4, 16), 0, f32x4{sum.m, sum.l, sum.t, 0.f});
      hand_publish();
    }
    __syncthreads();
    if (threadIdx.x == 0) s_last = hand_arrive(p.counters + row) == (uint32_t)(p.splits - 1);
    __syncthreads();
    if (!s_last) return;
    if (threadIdx.x == 0) hand_reset(p.counters + row);
    // lane by lane the sums of one split each, and the wave's lists, all on their way at once
    sum = Sums{-__builtin_inff(), 0.f, 0.f};
    if (lane < p.splits && (lane & (W - 1)) == part) {
      const f32x4 v = hand_load16(hand_buffer(p.sums + row * p.splits * 4, p.splits * 16), lane * 16);
      sum = Sums{v.x, v.y, v.z};
    }
    sum = join_lanes<1>(sum);
    best.list = 0;
    if (k > 0) {
      constexpr int MANY = kMaxSplits / WAVES;
      uint64_t* const lists = s_wait[wave];
#pragma unroll
      for (int i = 0; i < MANY; ++i) {
        const int s = part + i * W;
        lists[64 * i + lane] = s < p.splits && lane < k ? hand_load(p.keys + (row * p.splits + s) * k + lane) : (uint64_t)0;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 1
      for (int i = 0; part + i * W < p.splits; ++i) best.list = merged(best.list, lists[64 * i + 63 - lane]);
    }
    meet();
  }
  if (part != 0 || !real) return;

  // a NaN is in l even where it was never the maximum; nothing but -inf has l = 0
  const float log_l = __builtin_amdgcn_logf(sum.l);
  const float top = sum.m == -__builtin_inff() ? 0.f : sum.m;
  const auto logprob = [&](float v) {
    if (sum.l == 0.f) return v;
    return __builtin_fabsf(v) < kHuge ? (octaves(v, top) - log_l) * kLn2 : (v - top) - log_l * kLn2;
  };
  if (lane < k) {
    p.top_ids[row * k + lane] = (int32_t)~(uint32_t)best.list;
    p.top_logprobs[row * k + lane] = logprob(from_order((uint32_t)(best.list >> 32)));
  }
  if (lane == 0) {
    p.logprob[row] = token_there ? logprob(token_logit) : token_logit;
    p.entropy[row] = sum.l == 0.f ? 0.f : kLn2 * (log_l - sum.t / sum.l);
  }
}

struct Shape {
  int32_t splits;
  int64_t split_vectors;
  int32_t log_waves;  // waves of a row and split
};

// Waves of a row: enough rows fill the machine with one wave each (16 per compute unit); fewer take up
// to the four of a work-group, with two vectors a lane at least.  Long ones take several work-groups, which leave
// each wave kSplitTiles tiles (7 rows of 100003 fp32, 20 alternatives: 15.9 us so, 16.6 in half as many of
// eight waves), and where that makes no second work-group, one of eight waves (64 rows of 32000 fp16, 8
// alternatives: 13.0 us so, 14.5 of four, 13.1 of sixteen, 14.9 in two work-groups, 28.7 with one wave; 256 rows: 13.3,
// 14.9 of four, 30.3 with one).
Shape shape_of(int64_t rows, int64_t vocab, int per_vector, int32_t cus) {
  const int64_t vectors = ceil_div(vocab, per_vector) + 1;  // a row may begin inside a vector
  Shape s;
  int64_t want = vectors / (64 * kWaves * kVectors * kSplitTiles);
  if (rows > 0 && want > 2 * cus / rows) want = 2 * cus / rows;
  if (want > kMaxSplits) want = kMaxSplits;
  if (want < 1 || rows * 4 > BSG_KV_COUNTER_BYTES) want = 1;
  s.split_vectors = ceil_div(vectors, want);
  s.splits = (int32_t)ceil_div(vectors, s.split_vectors);
  const int most = s.splits > 1 ? kWaves : kMostWaves;
  s.log_waves = 0;
  while ((1 << s.log_waves) < most && (rows << s.log_waves) < 16 * (int64_t)cus && (128 << s.log_waves) < vectors)
    ++s.log_waves;
  return s;
}

int per_vector(int dtype) { return dtype == BSG_F32 ? 4 : 8; }

template <typename T>
void launch(const ScoreParams& p, dim3 grid, bool wide, hipStream_t st) {
  if (wide) hipLaunchKernelGGL((bsg_token_logprobs_kernel<T, kMostWaves>), grid, dim3(64 * kMostWaves), 0, st, p);
  else hipLaunchKernelGGL((bsg_token_logprobs_kernel<T, kWaves>), grid, dim3(64 * kWaves), 0, st, p);
}

int64_t workspace_bytes(const Shape& s, int64_t rows, int32_t k) {
  return s.splits <= 1 || rows == 0 ? 0 : BSG_KV_COUNTER_BYTES + rows * s.splits * (16 + 8 * (int64_t)k);
}

int check_sizes(int64_t rows, int64_t vocab, int32_t k, int dtype, int32_t cus) {
  if (dtype != BSG_F16 && dtype != BSG_BF16 && dtype != BSG_F32)
    return fail(BSG_ERR_DTYPE, "dtype=%d (0=fp16, 1=bf16, 2=fp32)", dtype);
  if (rows < 0 || vocab < 1 || k < 0 || k > vocab || cus < 1)
    return fail(BSG_ERR_ARG, "rows=%lld vocab=%lld k=%d cu_count=%d", (long long)rows, (long long)vocab, k, cus);
  if (k > kMaxK) return fail(BSG_ERR_UNSUPPORTED, "k=%d (at most %d)", k, kMaxK);
  if (vocab > 0x7fffffff || rows > 0x7fffffff)
    return fail(BSG_ERR_UNSUPPORTED, "rows=%lld vocab=%lld", (long long)rows, (long long)vocab);
  return BSG_OK;
}

}  // namespace

extern "C" int64_t bsg_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int32_t k, int dtype,
                                                      int32_t cu_count) {
  if (check_sizes(rows, vocab, k, dtype, cu_count)) return -1;
  return workspace_bytes(shape_of(rows, vocab, per_vector(dtype), cu_count), rows, k);
}

extern "C" int bsg_token_logprobs(const void* logits, int64_t row_stride, int64_t rows, int64_t vocab,
                                  const int32_t* tokens, int32_t k, float* logprob, float* entropy, int32_t* top_ids,
                                  float* top_logprobs, int dtype, void* ws, int64_t ws_bytes, int32_t cu_count,
                                  void* stream) {
  if (const int rc = check_sizes(rows, vocab, k, dtype, cu_count)) return rc;
  if (rows == 0) return BSG_OK;
  if (!logits || !tokens || !logprob || !entropy || (k > 0 && (!top_ids || !top_logprobs)))
    return fail(BSG_ERR_ARG, "null pointer (logits=%p tokens=%p logprob=%p entropy=%p top_ids=%p top_logprobs=%p)", logits,
                (const void*)tokens, (void*)logprob, (void*)entropy, (void*)top_ids, (void*)top_logprobs);
  if (!is_aligned(logits, dtype == BSG_F32 ? 4 : 2)) return fail(BSG_ERR_ALIGN, "logits must be aligned to their type");
  const Shape s = shape_of(rows, vocab, per_vector(dtype), cu_count);
  const int64_t need = workspace_bytes(s, rows, k);
  if (need > 0 && (!ws || ws_bytes < need))
    return fail(BSG_ERR_WORKSPACE, "workspace of %lld bytes, %lld needed", (long long)ws_bytes, (long long)need);
  if (need > 0 && !is_aligned(ws, 16)) return fail(BSG_ERR_ALIGN, "workspace must be 16-byte aligned");
  ScoreParams p;
  p.tokens = tokens;
  p.k = k;
  p.stride = row_stride;
  p.vocab = vocab;
  p.splits = s.splits;
  p.split_vectors = s.split_vectors;
  p.counters = (uint32_t*)ws;
  p.keys = need > 0 ? (uint64_t*)((uint8_t*)ws + BSG_KV_COUNTER_BYTES) : nullptr;
  p.sums = need > 0 ? (float*)(p.keys + rows * s.splits * k) : nullptr;
  const hipStream_t st = (hipStream_t)stream;
  const size_t es = dtype == BSG_F32 ? 4 : 2;
  // one launch takes 65535 work-groups of rows
  const bool wide = (1 << s.log_waves) > kWaves;
  const int64_t group = (wide ? kMostWaves : kWaves) >> s.log_waves, most = 65535 * group;
  p.log_waves = s.log_waves;
  for (int64_t r = 0; r < rows; r += most) {
    const int64_t n = rows - r < most ? rows - r : most;
    p.rows = (int32_t)n;
    p.x = (const uint8_t*)logits + r * row_stride * (int64_t)es;
    p.tokens = tokens + r;
    p.logprob = logprob + r;
    p.entropy = entropy + r;
    p.top_ids = k > 0 ? top_ids + r * k : nullptr;
    p.top_logprobs = k > 0 ? top_logprobs + r * k : nullptr;
    const dim3 grid((unsigned)s.splits, (unsigned)ceil_div(n, group));
    if (dtype == BSG_F16) launch<_Float16>(p, grid, wide, st);
    else if (dtype == BSG_BF16) launch<__bf16>(p, grid, wide, st);
    else launch<float>(p, grid, wide, st);
  }
  return launch_status("bsg_token_logprobs");
}
