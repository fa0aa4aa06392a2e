// verify.hip — which drafted tokens a target model accepts, and the token that follows them (include/bsgdraft.h,
// bsgdraft_slots.h).
//
// Answers are whole numbers next to borders: a number u against a ratio of probabilities, and the first running sum past
// u of the whole.  So weights w = 2^((x - m) k), k = log2(e) / temperature, and their sums are 64-bit.  2^t is
// 2^n times a polynomial of the 9th degree in f, t = n + f, |f| <= 1/2, which interpolates 2^f in the Chebyshev points of
// that interval (relative error 2^-45.6).
//
// First launch: of the rows of nodes that have children a wave has kPiece logits in registers and leaves their maximum
// and the sum of their weights against it (or, greedy, where the first maximum is).  Second launch: the work-groups
// of a sequence each put the rows together and walk the tree (a node in each lane; nodes in order, each asked if its
// parent is the last accepted one); then each makes the sums of some pieces of what is left of the last row, and the last
// to arrive draws the new token, first a piece, then a number of it.
//
// Of a row without draft_logits the walk only asks on which side of a number its sum lies, so that the first launch adds its
// weights in 32 bits, kNear off at most; where a number is as near as that to its border the wave adds the row again in
// 64.  Against draft_logits the last row's sums are wanted exactly, and both are 64-bit from the start.

#include "bsgdraft_slots.h"
#include "draft_tree.hpp"

using namespace bsgk;

namespace {

// Logits of a wave.  512, 1024, 2048, both launches, us: 64 chains of 5 38, 33, 34; 64 trees of 16 36, 30, 31; 8 of 16 18, 17, 20.
constexpr int kPiece = 1024;
constexpr int kWaves = 4;     // of a work-group
constexpr int kMostVocab = 1 << 20;
constexpr double kLog2e = 1.4426950408889634;
// The 32-bit sum of a row: a weight of t octaves is off by 0.7 x 3 |t| 2^-24 (the difference, k, their product) and 2^-22 of
// itself; |t|, averaged by the weights, is at most the logarithm of the vocabulary, 20.  A lane's sum of 16 numbers adds 2^-20.
constexpr double kNear = 0x1p-17;

struct Piece {  // of a row
  double sum;   // of its weights; NaN: a logit is NaN or +inf
  float top;
  int32_t at;   // of the first maximum
};

struct VerifyParams {
  const void* x[2];  // the target's logits, the drafts'
  int64_t stride[2];
  int64_t vocab, tokens;
  const int32_t* ids;
  const float* uniforms;
  const int32_t* parents;
  const int32_t* cu;
  const int32_t* slots;  // below 0: the sequence takes no part
  const float* temperatures;
  float temperature;
  int32_t rows, max_new, pieces, groups, drafts;  // pieces of a row, work-groups of a row
  int32_t* accepted;
  int32_t* path;
  int32_t* out;
  uint32_t* counters;  // [rows]: of the second launch
  Piece* stats;        // [tokens][1 + drafts][pieces]
  Piece* last;         // [rows][pieces], of the last row
};

// The weight of a logit against a maximum: 2^((x - top) k), 0 far below and for -inf (and NaN, which its row is known by).
__device__ __forceinline__ double weight(float x, float top, double k) {
  const double t = __builtin_fmax(((double)x - (double)top) * k, -1100.0);
  const double n = __builtin_rint(t), f = t - n;
  double y = 1.0205905413765595e-07;
  y = __builtin_fma(y, f, 1.325964524488711e-06);
  y = __builtin_fma(y, f, 1.5252672924850737e-05);
  y = __builtin_fma(y, f, 0.0001540343375125101);
  y = __builtin_fma(y, f, 0.0013333558200794592);
  y = __builtin_fma(y, f, 0.009618129193934313);
  y = __builtin_fma(y, f, 0.05550410866465167);
  y = __builtin_fma(y, f, 0.2402265069564034);
  y = __builtin_fma(y, f, 0.6931471805599462);
  y = __builtin_fma(y, f, 1.0000000000000135);
  return __builtin_ldexp(y, (int)n);
}

template <typename T>
struct Logit;
template <>
struct Logit<float> {
  static constexpr int PER = 4;  // of 16 bytes
  static __device__ __forceinline__ float of(const u32x4& v, int e) { return as_float(v[e]); }
  static __device__ __forceinline__ float one(const void* x, int64_t at) { return ((const float*)x)[at]; }
};
template <>
struct Logit<_Float16> {
  static constexpr int PER = 8;
  static __device__ __forceinline__ float of(const u32x4& v, int e) { return e & 1 ? high_half<_Float16>(v[e >> 1]) : low_half<_Float16>(v[e >> 1]); }
  static __device__ __forceinline__ float one(const void* x, int64_t at) { return (float)((const _Float16*)x)[at]; }
};
template <>
struct Logit<__bf16> {
  static constexpr int PER = 8;
  static __device__ __forceinline__ float of(const u32x4& v, int e) { return e & 1 ? high_half<__bf16>(v[e >> 1]) : low_half<__bf16>(v[e >> 1]); }
  static __device__ __forceinline__ float one(const void* x, int64_t at) { return as_float((uint32_t)((const uint16_t*)x)[at] << 16); }
};

// Numbers of a row in registers.  A row is cut at addresses that 16 bytes divide, so that every load is whole (the granules in
// which it begins and ends are read whole); `shift` is how many numbers of the first granule lie before the row.  What
// lies outside the row is -inf.
template <typename T>
__device__ __forceinline__ int shift_of(const void* x, int64_t row_at) {
  return (int)(((uintptr_t)((const T*)x + row_at) & 15) / sizeof(T));
}
template <typename T, int BYTES>
struct Numbers {
  typedef T vec __attribute__((ext_vector_type(Logit<T>::PER)));
  static constexpr int PER = Logit<T>::PER, VECTORS = BYTES / 16, N = PER * VECTORS;
  u32x4 v[VECTORS];
  // f(number of the vector, vector) for one after the other, in a loop: a wave comes by here once or twice, and code
  // that is not in the instruction cache yet costs more than the loop.  OFTEN: a compute unit has many such waves, and
  // the loop's moves cost more (64 chains, first launch: 17 against 18 us).
  template <bool OFTEN = false, typename F>
  __device__ __forceinline__ void each(const F& f) {
    if constexpr (OFTEN) {
#pragma unroll
      for (int k = 0; k < VECTORS; ++k) f(k, v[k]);
      return;
    }
#pragma unroll 1
    for (int k = 0; k < VECTORS; ++k) {
      u32x4 first = v[0];
      f(k, first);
#pragma unroll
      for (int i = 0; i + 1 < VECTORS; ++i) v[i] = v[i + 1];
      v[VECTORS - 1] = first;
    }
  }
  // Vector k from number at(k) of a row on.  shift: the cut's, which is the row's own but where it goes beside another row.
  template <typename At>
  __device__ __forceinline__ void load(const void* x, int64_t row_at, int n, int shift, bool inside, const At& at) {
    const T* const row = (const T*)x + row_at;
    const bool own = shift_of<T>(x, row_at) == shift;
    // all loads before one is looked at; what lies outside loads the first granule
    if (own) {
#pragma unroll
      for (int k = 0; k < VECTORS; ++k) v[k] = *(const u32x4*)(row + (at(k) < n ? at(k) : -shift));
      if (inside) return;
    }
    each([&](int k, u32x4& a) {
      vec w = __builtin_bit_cast(vec, a);
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const bool in = at(k) + e >= 0 && at(k) + e < n;
        if (!own) w[e] = row[in ? at(k) + e : 0];
        w[e] = in ? w[e] : (T)-__builtin_inff();
      }
      a = __builtin_bit_cast(u32x4, w);
    });
  }
  // The number that the row has at `place` weighs nothing any more, if it is one of the lane's.
  template <typename At>
  __device__ __forceinline__ void drop(int place, const At& at) {
    each([&](int k, u32x4& a) {
      vec w = __builtin_bit_cast(vec, a);
#pragma unroll
      for (int e = 0; e < PER; ++e) w[e] = at(k) + e == place ? (T)-__builtin_inff() : w[e];
      a = __builtin_bit_cast(u32x4, w);
    });
  }
};
// A wave's piece: vector k of lane l from number (64 k + l) PER of it on.
template <typename T>
struct PieceOf : Numbers<T, (int)(kPiece / 64 * sizeof(T))> {
  static constexpr int PER = Logit<T>::PER;
  __device__ __forceinline__ void load(const void* x, int64_t row_at, int64_t vocab, int shift, int piece, int lane) {
    const int first = piece * kPiece - shift, n = (int)vocab;
    Numbers<T, (int)(kPiece / 64 * sizeof(T))>::load(x, row_at, n, shift, first >= 0 && first + kPiece <= n,
                                                     [&](int k) { return first + (64 * k + lane) * PER; });
  }
  __device__ __forceinline__ void drop(int place, int shift, int piece, int lane) {
    Numbers<T, (int)(kPiece / 64 * sizeof(T))>::drop(place, [&](int k) { return piece * kPiece - shift + (64 * k + lane) * PER; });
  }
};
// A wave's share of the piece that the new token is drawn from: lane l has the numbers 8 l .. 8 l + 7 of it.
constexpr int kShare = 512;
template <typename T>
struct ShareOf : Numbers<T, (int)(kShare / 64 * sizeof(T))> {
  static constexpr int PER = Logit<T>::PER, N = kShare / 64;
  __device__ __forceinline__ void load(const void* x, int64_t row_at, int64_t vocab, int shift, int first, int lane) {
    const int n = (int)vocab;
    Numbers<T, (int)(kShare / 64 * sizeof(T))>::load(x, row_at, n, shift, first >= 0 && first + kShare <= n,
                                                       [&](int k) { return first + lane * N + k * PER; });
  }
  __device__ __forceinline__ void drop(int place, int first, int lane) {
    Numbers<T, (int)(kShare / 64 * sizeof(T))>::drop(place, [&](int k) { return first + lane * N + k * PER; });
  }
  __device__ __forceinline__ float get(int i) const { return Logit<T>::of(this->v[i / PER], i % PER); }
};

template <int X>
__device__ __forceinline__ double lane_xor64(double v) {
  return __builtin_bit_cast(double, lane_xor<X>(__builtin_bit_cast(uint64_t, v)));
}
template <int X>
__device__ __forceinline__ double wave_sum(double v) {
  v += lane_xor64<X>(v);
  if constexpr (X > 1) v = wave_sum<X / 2>(v);
  return v;
}
template <int X>
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, lane_xor<X>(v));
  if constexpr (X > 1) v = wave_max<X / 2>(v);
  return v;
}
template <int X>
__device__ __forceinline__ int wave_min(int v) {
  const int o = (int)lane_xor<X>((uint32_t)v);
  v = o < v ? o : v;
  if constexpr (X > 1) v = wave_min<X / 2>(v);
  return v;
}
// Sum over the lanes up to this one.
__device__ __forceinline__ double wave_scan(double v, int lane) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const double o = __shfl_up(v, m);
    if (lane >= m) v += o;
  }
  return v;
}

// A sequence, as every wave of it sees it.
struct Tree {
  int64_t from;
  int count;
  float temperature;
  int parent;  // of node `lane`
};
__device__ __forceinline__ Tree tree_of(const VerifyParams& p, int row, int lane) {
  Tree t;
  t.from = (int64_t)row * p.max_new;
  int64_t to = t.from + p.max_new;
  if (p.cu) t.from = p.cu[row], to = p.cu[row + 1];
  t.temperature = p.temperatures ? p.temperatures[row] : p.temperature;
  // whose inverse is a 32-bit number other than 0, and infinity: no product with it is NaN
  if (t.temperature > 0.f) t.temperature = fminf(fmaxf(t.temperature, 0x1p-126f), 0x1.fffffep127f);
  const bool fine = t.from >= 0 && t.from < to && to <= p.tokens && !(p.slots && p.slots[row] < 0);
  t.count = !fine ? 0 : to - t.from < p.max_new ? (int)(to - t.from) : p.max_new;
  t.parent = load_parent(p.parents, t.from, t.count, lane);
  return t;
}
// The nodes that have children.
__device__ __forceinline__ uint64_t inner_of(const Tree& t) {
  uint64_t v = t.parent >= 0 ? 1ull << t.parent : 0;
  v |= lane_xor<1>(v), v |= lane_xor<2>(v), v |= lane_xor<4>(v);
  v |= lane_xor<8>(v), v |= lane_xor<16>(v), v |= lane_xor<32>(v);
  return v;
}

// What a piece is to its row: its maximum, the sum of its weights against that, and greedy the place of the first
// maximum.  first: the place of the piece's first number.
template <bool OFTEN, typename T>
__device__ __forceinline__ Piece piece_of(PieceOf<T>& x, bool greedy, bool exact, double k, int first, int lane) {
  constexpr int PER = PieceOf<T>::PER;
  bool bad = false;
  float top = -__builtin_inff();
  x.template each<OFTEN>([&](int, u32x4& v) {
#pragma unroll
    for (int e = 0; e < PER; ++e) top = fmaxf(top, Logit<T>::of(v, e)), bad = bad || !(Logit<T>::of(v, e) < __builtin_inff());
  });
  Piece mine = {0.0, wave_max<32>(top), 0x7fffffff};
  if (greedy) {
    x.template each<OFTEN>([&](int i, u32x4& v) {
#pragma unroll
      for (int e = PER - 1; e >= 0; --e)
        if (Logit<T>::of(v, e) == mine.top && first + (64 * i + lane) * PER + e < mine.at) mine.at = first + (64 * i + lane) * PER + e;
    });
    mine.at = wave_min<32>(mine.at);
  } else if (exact) {
    x.template each<OFTEN>([&](int, u32x4& v) {
#pragma unroll
      for (int e = 0; e < PER; ++e) mine.sum += weight(Logit<T>::of(v, e), mine.top, k);
    });
    mine.sum = wave_sum<32>(mine.sum);
  } else {
    // a piece of nothing but -inf has no maximum to be weighed against
    const float by = (float)k, from = mine.top == -__builtin_inff() ? 0.f : mine.top;
    float sum = 0.f;
    x.template each<OFTEN>([&](int, u32x4& v) {
#pragma unroll
      for (int e = 0; e < PER; ++e) sum += __builtin_amdgcn_exp2f((Logit<T>::of(v, e) - from) * by);
    });
    mine.sum = wave_sum<32>((double)sum);
  }
  if (__any(bad)) mine.sum = __builtin_nan("");
  return mine;
}

// The rows of the nodes that have children, by pieces: of a sequence's the blockIdx.y-th, and every gridDim.y-th from there.
// 64 chains of up to 5 drawn drafts, 32000 fp16 logits of two models: 17 us, of which the 64-bit weights are some 12 (18
// instructions each, the sum's among them, all at the rate of a fused multiply-add); 64 trees of up to 16 nodes: 13 us with
// 32-bit weights, 21 with 64-bit ones.
template <typename T>
__global__ __launch_bounds__(64 * kWaves) void bsg_verify_rows_kernel(VerifyParams p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int which = blockIdx.x / p.groups, piece = (blockIdx.x - which * p.groups) * kWaves + wave;
  const Tree t = tree_of(p, blockIdx.z, lane);
  const bool greedy = !(t.temperature > 0.f);
  if (piece >= p.pieces || (greedy && which)) return;
  uint64_t left = inner_of(t);
  for (int skip = blockIdx.y; left; skip = gridDim.y - 1) {
    for (; skip > 0 && left; --skip) left &= left - 1;
    if (!left) return;
    const int node = __builtin_amdgcn_readfirstlane(__builtin_ctzll(left));
    left &= left - 1;
    const int64_t at = (t.from + node) * p.stride[which];
    // a draft's row is cut as the target's beside it is, so that of equal rows the sums are equal to the last bit
    const int shift = shift_of<T>(p.x[0], (t.from + node) * p.stride[0]);
    PieceOf<T> x;
    x.load(p.x[which], at, p.vocab, shift, piece, lane);
    const Piece mine = piece_of<true, T>(x, greedy, p.drafts != 0, kLog2e / (double)t.temperature, piece * kPiece - shift, lane);
    if (lane == 0) p.stats[((t.from + node) * (1 + p.drafts) + which) * p.pieces + piece] = mine;
  }
}

__device__ __forceinline__ double read_lane(double v, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)b, lane), hi = __builtin_amdgcn_readlane((int)(b >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// The sequence's answer: the accepted nodes (a bit for each), and the new token.  id: of node `lane`.  A wave's work.
__device__ __forceinline__ void answer(const VerifyParams& p, int row, uint64_t taken, int id, int token, int lane) {
  const int count = __builtin_popcountll(taken);
  int32_t* const path = p.path + (int64_t)row * p.max_new;
  int32_t* const out = p.out + (int64_t)row * p.max_new;
  const int place = __builtin_popcountll(taken & ((1ull << lane) - 1));
  const bool mine = taken >> lane & 1;
  if (mine) path[place] = lane;
  if (mine && place > 0) out[place - 1] = id;
  if (lane == 0 && count > 0) out[count - 1] = token;
  for (int i = count + lane; i < p.max_new; i += 64) path[i] = -1, out[i] = -1;
  if (lane == 0) p.accepted[row] = count;
}

// The piece of a row that `u` of its whole falls into: the first one whose running sum passes that, the last one of any
// weight if none does, -1 without any.  load(i) gives piece i, weighed against its own maximum, or, WEIGHED,
// against the row's.  A lane has `each` pieces that follow each other.
struct Picked {
  int piece;
  float top;             // of the row
  double whole, before;  // sums of the row, and of the pieces before
};
template <bool WEIGHED, typename Load>
__device__ __forceinline__ Picked pick_piece(int pieces, double u, double k, int lane, const Load& load) {
  const int each = (pieces + 63) / 64;
  Picked r = {-1, -__builtin_inff(), 0.0, 0.0};
  Piece v = {0.0, -__builtin_inff(), 0};
  if constexpr (!WEIGHED) {
    for (int i = 0; i < each; ++i)
      if (lane * each + i < pieces) v = load(lane * each + i), r.top = fmaxf(r.top, v.top);
    r.top = wave_max<32>(r.top);
  }
  const auto sum_of = [&](int i) {
    if (lane * each + i >= pieces) return 0.0;
    if (WEIGHED || each > 1) v = load(lane * each + i);
    return WEIGHED || v.sum != v.sum ? v.sum : v.sum * weight(v.top, r.top, k);
  };
  double mine = 0.0;
  for (int i = 0; i < each; ++i) mine += sum_of(i);
  const double upto = wave_scan(mine, lane);
  r.whole = read_lane(upto, 63);
  const double goal = u * r.whole;
  const uint64_t past = __ballot(upto > goal && mine > 0.0), some = __ballot(mine > 0.0);
  if (!some) return r;
  const int at = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
  double run = upto - mine, before = run;
  int hit = -1;
  if (each == 1) {
    hit = 0;
  } else {
    bool found = false;
    for (int i = 0; i < each; ++i) {
      const double w = sum_of(i);
      if (!found && w > 0.0) hit = i, before = run, found = run + w > goal;
      run += w;
    }
  }
  r.piece = at * each + __builtin_amdgcn_readlane(hit, at), r.before = read_lane(before, at);
  return r;
}

// The place in its piece of the first number whose running sum, from `before` on, passes `goal`; the last one of any weight if
// none does; -1 without any.  A work-group's work: each wave has a share of the piece, or nothing, a lane N consecutive numbers.
template <int N>
__device__ __forceinline__ int pick_number(const double (&w)[N], double before, double goal, int lane, int wave) {
  __shared__ double s_sum[kWaves];
  __shared__ int2 s_hit[kWaves];  // the first number past the goal, the last of any weight
  double sum = 0.0;
  int any = -1;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    sum += w[i];
    if (w[i] > 0.0) any = i;
  }
  const double scan = wave_scan(sum, lane);
  if (lane == 63) s_sum[wave] = scan;
  __syncthreads();
  for (int i = 0; i < wave; ++i) before += s_sum[i];
  const double upto = before + scan;
  double run = upto - sum;
  int hit = -1;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    run += w[i];
    if (hit < 0 && w[i] > 0.0 && run > goal) hit = i;
  }
  // the lane's own sum may be short of the scan's by a last bit
  if (hit < 0 && any >= 0 && upto > goal) hit = any;
  const uint64_t past = __ballot(hit >= 0), some = __ballot(any >= 0);
  if (lane == 0) s_hit[wave] = make_int2(-1, -1);
  if (past && lane == __builtin_ctzll(past)) s_hit[wave].x = wave * kShare + lane * N + hit;
  if (some && lane == 63 - __builtin_clzll(some)) s_hit[wave].y = wave * kShare + lane * N + any;
  __syncthreads();
  int at = -1;
  for (int i = 0; i < kWaves; ++i)
    if (s_hit[i].y >= 0) at = s_hit[i].y;
  for (int i = kWaves - 1; i >= 0; --i)
    if (s_hit[i].x >= 0) at = s_hit[i].x;
  return at;
}

__device__ __forceinline__ Piece load_piece(const Piece* at) {
  Piece v;
  v.sum = __builtin_bit_cast(double, hand_load((const uint64_t*)at));
  const uint64_t b = hand_load((const uint64_t*)at + 1);
  v.top = as_float((uint32_t)b), v.at = (int32_t)(b >> 32);
  return v;
}
__device__ __forceinline__ void store_piece(Piece* at, const Piece& v) {
  hand_store((uint64_t*)at, __builtin_bit_cast(uint64_t, v.sum));
  hand_store((uint64_t*)at + 1, (uint64_t)(uint32_t)v.at << 32 | __builtin_bit_cast(uint32_t, v.top));
}

// A row's maximum, the sum of its weights against it and the place of the first maximum, from its pieces, by a segment of
// `seg` lanes (16, 32 or 64), each of which gets them.
struct Row {
  double total;
  float top;
  int32_t at;
};
template <typename Load>
__device__ __forceinline__ Row row_of(int pieces, double k, int seg, int lane, const Load& load) {
  Row r = {0.0, -__builtin_inff(), 0x7fffffff};
  const int sub = lane & (seg - 1);
  Piece v = {0.0, -__builtin_inff(), 0x7fffffff};
  for (int c = sub; c < pieces; c += seg) {
    v = load(c);
    r.top = fmaxf(r.top, v.top);
  }
  if (seg > 32) r.top = fmaxf(r.top, lane_xor<32>(r.top));
  if (seg > 16) r.top = fmaxf(r.top, lane_xor<16>(r.top));
  r.top = wave_max<8>(r.top);
  for (int c = sub; c < pieces; c += seg) {
    if (pieces > seg) v = load(c);
    if (v.top == r.top && v.at < r.at) r.at = v.at;
    r.total += v.sum == v.sum ? v.sum * weight(v.top, r.top, k) : v.sum;
  }
  const auto join = [&](double total, int32_t at) { r.total += total, r.at = at < r.at ? at : r.at; };
  if (seg > 32) join(lane_xor64<32>(r.total), (int32_t)lane_xor<32>((uint32_t)r.at));
  if (seg > 16) join(lane_xor64<16>(r.total), (int32_t)lane_xor<16>((uint32_t)r.at));
  r.total = wave_sum<8>(r.total), r.at = wave_min<8>(r.at);
  return r;
}

// A chain of waits bounds it, of which none is long: the tree, the rows' pieces, the walk, a piece of the last row, the meeting
// of the work-groups, the piece and the number that are drawn.  64 chains 15 us, 64 trees 16, of 32000 logits; greedy 9.
template <typename T>
__global__ __launch_bounds__(64 * kWaves) void bsg_verify_walk_kernel(VerifyParams p) {
  constexpr int PER = PieceOf<T>::PER, N = ShareOf<T>::N;
  __shared__ double s_total[2][BSG_TREE_NODES];
  __shared__ float s_top[2][BSG_TREE_NODES];
  __shared__ int32_t s_at[BSG_TREE_NODES];
  __shared__ uint32_t s_last;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = blockIdx.y, group = blockIdx.x;
  const Tree t = tree_of(p, row, lane);
  if (t.count == 0) {
    if (group == 0 && wave == 0) answer(p, row, 0, -1, -1, lane);
    return;
  }
  const bool greedy = !(t.temperature > 0.f), drafts = p.drafts != 0 && !greedy;
  const double k = greedy ? 1.0 : kLog2e / (double)t.temperature;
  // node `lane`: its token, its number, and the token's logits in its parent's rows
  const int id = lane < t.count ? p.ids[t.from + lane] : -1;
  const double u = lane < t.count ? (double)p.uniforms[t.from + lane] : 0.0;
  const int up = t.parent < 0 ? 0 : t.parent;
  const bool known = t.parent >= 0 && id >= 0 && id < p.vocab;
  float x0 = 0.f, x1 = 0.f;
  if (known && !greedy) {
    x0 = Logit<T>::one(p.x[0], (t.from + up) * p.stride[0] + id);
    if (drafts) x1 = Logit<T>::one(p.x[1], (t.from + up) * p.stride[1] + id);
  }

  const uint64_t inner = inner_of(t);
  const auto stats = [&](int node, int which) { return p.stats + ((t.from + node) * (1 + p.drafts) + which) * p.pieces; };
  {
    const int seg = p.pieces <= 16 ? 16 : p.pieces <= 32 ? 32 : 64, each = 64 / seg;
    const int rows = __builtin_popcountll(inner);
    for (int i0 = wave * each; i0 < (drafts ? 2 * rows : rows); i0 += kWaves * each) {
      const int i = i0 + lane / seg, which = i >= rows;
      // the (i or i - rows)-th of the nodes that have children
      int nth = which ? i - rows : i, node = 0;
      for (uint64_t m = inner; m && nth >= 0; m &= m - 1, --nth) node = __builtin_ctzll(m);
      const bool on = i < (drafts ? 2 * rows : rows);
      const Piece* const at = stats(on ? node : __builtin_ctzll(inner), on ? which : 0);
      const Row r = row_of(p.pieces, k, seg, lane, [&](int c) { return at[c]; });
      if (on && (lane & (seg - 1)) == 0) {
        s_total[which][node] = r.total, s_top[which][node] = r.top;
        if (!which) s_at[node] = r.at;
      }
    }
  }
  __syncthreads();

  // Of a node's row, against its maximum: by each wave for itself, seldom.
  const auto exact_total = [&](int node) {
    const int64_t from = (t.from + node) * p.stride[0];
    const int off = shift_of<T>(p.x[0], from);
    double sum = 0.0;
#pragma unroll 1
    for (int c = 0; c < p.pieces; ++c) {
      PieceOf<T> x;
      x.load(p.x[0], from, p.vocab, off, c, lane);
      x.each([&](int, u32x4& v) {
#pragma unroll
        for (int e = 0; e < PER; ++e) sum += weight(Logit<T>::of(v, e), s_top[0][node], k);
      });
    }
    return wave_sum<32>(sum);
  };

  // every wave walks
  double mine = 0.0, theirs = 0.0;
  if (known && !greedy) {
    mine = weight(x0, s_top[0][up], k);
    if (drafts) mine /= s_total[0][up], theirs = weight(x1, s_top[1][up], k) / s_total[1][up];
  }
  int at = 0;
  uint64_t taken = 1, refused = 0;  // refused: the rejected children of `at`, of each token one
  double out = 0.0;                 // their weights
  double total = inner != 0 ? s_total[0][0] : 0.0;
  bool exact = drafts;              // total is
  for (uint64_t left = ~1ull;;) {
    const uint64_t asked = left & __ballot(t.parent >= 0 && t.parent == at);
    if (!asked) break;
    const int j = __builtin_ctzll(asked);
    left = j == 63 ? 0 : left & ~0ull << (j + 1);
    const bool same = (refused & __ballot(id == __builtin_amdgcn_readlane(id, j))) != 0;  // has no weight left
    const double u_j = read_lane(u, j), w_j = read_lane(mine, j);
    bool ok = (__ballot(known) >> j & 1) != 0 && !same;
    if (greedy) {
      ok = ok && __builtin_amdgcn_readlane(id, j) == s_at[at] && total == total && s_top[0][at] > -__builtin_inff();
    } else if (drafts) {
      ok = ok && u_j * read_lane(theirs, j) < w_j;
    } else if (ok) {
      if (!exact && __builtin_fabs(u_j * (total - out) - w_j) <= kNear * total * u_j) {
        total = exact_total(at), exact = true;
      }
      ok = u_j * (total - out) < w_j;
    }
    if (ok) {
      at = j, taken |= 1ull << j, refused = 0, out = 0.0;
      total = inner >> j & 1 ? s_total[0][j] : 0.0, exact = drafts;
    } else if (!same) {
      refused |= 1ull << j, out += w_j;
    }
  }

  const bool leaf = (inner >> at & 1) == 0, residual = drafts && refused != 0;
  float top = leaf ? 0.f : s_top[0][at];
  // known by now: greedy of a row that the first launch had; none of a row that has no probabilities
  if (!leaf && (greedy || !(total > 0.0))) {
    const bool some = greedy && total == total && top > -__builtin_inff();
    if (group == 0 && wave == 0) answer(p, row, taken, id, some ? s_at[at] : -1, lane);
    return;
  }

  // what is left of the last row: the row without the rejected tokens, or what it has over its drafts
  const int64_t x_at = (t.from + at) * p.stride[0], y_at = (t.from + at) * p.stride[1];
  const int shift = shift_of<T>(p.x[0], x_at);
  const double by[2] = {1.0 / total, residual ? 1.0 / s_total[1][at] : 0.0};
  const float y_top = residual ? s_top[1][at] : 0.f;
  const auto surplus = [&](double x, double y) {
#pragma clang fp contract(off)  // each product rounded: a q that is p leaves nothing of it
    return __builtin_fmax(x * by[0] - y * by[1], 0.0);
  };
  Piece* const last = p.last + (int64_t)row * p.pieces;
  int token = -1;
  for (bool again = false;; again = true) {
    // its own piece; again: all of them
    for (int piece = again ? wave : group * kWaves + wave; piece < p.pieces; piece += again ? kWaves : p.pieces) {
      PieceOf<T> x;
      x.load(p.x[0], x_at, p.vocab, shift, piece, lane);
      Piece v = {0.0, 0.f, 0};
      if (residual) {
        PieceOf<T> y;
        y.load(p.x[1], y_at, p.vocab, shift, piece, lane);
        x.each([&](int, u32x4& a) {
          const u32x4 b = y.v[0];
#pragma unroll
          for (int e = 0; e < PER; ++e) v.sum += surplus(weight(Logit<T>::of(a, e), top, k), weight(Logit<T>::of(b, e), y_top, k));
#pragma unroll
          for (int i = 0; i + 1 < PieceOf<T>::VECTORS; ++i) y.v[i] = y.v[i + 1];
        });
        v.sum = wave_sum<32>(v.sum);
      } else {
        for (uint64_t m = refused; m; m &= m - 1) x.drop(__builtin_amdgcn_readlane(id, __builtin_ctzll(m)), shift, piece, lane);
        v = piece_of<false, T>(x, greedy, true, k, piece * kPiece - shift, lane);
      }
      if (lane == 0) store_piece(last + piece, v);
    }
    hand_publish();
    __syncthreads();
    if (!again) {
      if (threadIdx.x == 0) s_last = hand_arrive(p.counters + row) == (uint32_t)(p.groups - 1);
      __syncthreads();
      if (!s_last) return;
      if (threadIdx.x == 0) hand_reset(p.counters + row);
    }
    if (greedy) {
      const Row r = row_of(p.pieces, k, 64, lane, [&](int c) { return load_piece(last + c); });
      if (r.total == r.total && r.top > -__builtin_inff()) token = r.at;
      break;
    }
    const double draw = read_lane(u, 0);
    bool over = residual;  // something is left of the row over its drafts; else from the row
    Picked c;
    if (residual) c = pick_piece<true>(p.pieces, draw, k, lane, [&](int i) { return load_piece(last + i); });
    over = residual && c.whole > 0.0;
    if (!over) {
      const Piece* const own = stats(at, 0);
      c = pick_piece<false>(p.pieces, draw, k, lane, [&](int i) { return residual ? own[i] : load_piece(last + i); });
      top = c.top;
    }
    if (!(c.whole > 0.0) && refused != 0 && !residual) {
      // the rejected tokens had all of the row's weight: the new token is drawn from all of it, of which only this work-group is
      // still here
      refused = 0;
      __syncthreads();  // every wave has read the sums, which are alike for all
      continue;
    }
    if (c.whole > 0.0) {
      double w[N];
      const int first = c.piece * kPiece + wave * kShare - shift;
      if (wave < kPiece / kShare) {
        ShareOf<T> x, y;
        x.load(p.x[0], x_at, p.vocab, shift, first, lane);
        if (over) y.load(p.x[1], y_at, p.vocab, shift, first, lane);
        if (!residual)
          for (uint64_t m = refused; m; m &= m - 1) x.drop(__builtin_amdgcn_readlane(id, __builtin_ctzll(m)), first, lane);
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = weight(x.get(i), top, k);
        if (over) {
#pragma unroll
          for (int i = 0; i < N; ++i) w[i] = surplus(w[i], weight(y.get(i), y_top, k));
        }
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = 0.0;
      }
      const int in_piece = pick_number(w, c.before, draw * c.whole, lane, wave);
      if (in_piece >= 0) token = in_piece + c.piece * kPiece - shift;
    }
    break;
  }
  if (wave == 0) answer(p, row, taken, id, token, lane);
}

struct Layout {
  int64_t pieces, stats, last, bytes;  // of a row; where they lie in the workspace
};
Layout layout_of(int64_t tokens, int32_t rows, int64_t vocab, int32_t drafts) {
  Layout l;
  l.pieces = ceil_div(vocab + 7, kPiece);  // with up to 7 numbers of the first granule before the row
  l.stats = BSG_KV_COUNTER_BYTES;
  l.last = l.stats + tokens * (1 + drafts) * l.pieces * (int64_t)sizeof(Piece);
  l.bytes = l.last + rows * l.pieces * (int64_t)sizeof(Piece);
  return l;
}

int check_sizes(int64_t tokens, int32_t rows, int64_t vocab, int32_t max_new, int dtype) {
  if (dtype != BSG_F16 && dtype != BSG_BF16 && dtype != BSG_F32) return fail(BSG_ERR_DTYPE, "dtype=%d (0=fp16, 1=bf16, 2=fp32)", dtype);
  if (tokens < 0 || rows < 0 || vocab < 1 || max_new < 0 || tokens > 0x7fffffff)
    return fail(BSG_ERR_ARG, "tokens=%lld rows=%d vocab=%lld max_new=%d", (long long)tokens, rows, (long long)vocab, max_new);
  if (max_new > BSG_TREE_NODES) return fail(BSG_ERR_UNSUPPORTED, "%d nodes in a tree (at most %d)", max_new, BSG_TREE_NODES);
  if (vocab > kMostVocab) return fail(BSG_ERR_UNSUPPORTED, "vocab=%lld (at most %d)", (long long)vocab, kMostVocab);
  if (rows > BSG_KV_COUNTER_BYTES / 4) return fail(BSG_ERR_UNSUPPORTED, "%d sequences (at most %d)", rows, BSG_KV_COUNTER_BYTES / 4);
  return BSG_OK;
}

template <typename T>
void launch(const VerifyParams& p, hipStream_t st) {
  if (p.max_new > 1) {  // else no node has children
    // Most of a large tree's nodes have no children, and their work-groups would only come and go: work-groups for all nodes, for
    // half of them, us: 64 trees of 16 34, 30; 8 of 64 37, 34; 8 of 8 20.4, 20.7.
    const int at_once = p.max_new <= 8 ? p.max_new - 1 : p.max_new / 2;
    const dim3 grid((unsigned)(p.groups * (1 + p.drafts)), (unsigned)at_once, (unsigned)p.rows);
    hipLaunchKernelGGL((bsg_verify_rows_kernel<T>), grid, dim3(64 * kWaves), 0, st, p);
  }
  hipLaunchKernelGGL((bsg_verify_walk_kernel<T>), dim3((unsigned)p.groups, (unsigned)p.rows), dim3(64 * kWaves), 0, st, p);
}

}  // namespace

extern "C" int64_t bsg_verify_drafts_workspace_bytes(int64_t tokens, int32_t rows, int64_t vocab, int32_t max_new, int dtype,
                                                     int32_t drafts) {
  if (check_sizes(tokens, rows, vocab, max_new, dtype)) return -1;
  return layout_of(tokens, rows, vocab, drafts != 0).bytes;
}

extern "C" int bsg_verify_drafts(const void* logits, int64_t logits_stride, const void* draft_logits, int64_t draft_stride,
                                 int64_t tokens, int64_t vocab, const int32_t* token_ids, const float* uniforms,
                                 const int32_t* parents, const int32_t* cu, int32_t rows, int32_t max_new,
                                 float temperature, const float* temperatures, int32_t* accepted, int32_t* path,
                                 int32_t* out_tokens, int dtype, void* ws, int64_t ws_bytes, void* stream) {
  return bsg_verify_drafts_slots(logits, logits_stride, draft_logits, draft_stride, tokens, vocab, token_ids, uniforms, parents,
                                 cu, nullptr, rows, max_new, temperature, temperatures, accepted, path, out_tokens, dtype, ws,
                                 ws_bytes, stream);
}

extern "C" int bsg_verify_drafts_slots(const void* logits, int64_t logits_stride, const void* draft_logits,
                                       int64_t draft_stride, int64_t tokens, int64_t vocab, const int32_t* token_ids,
                                       const float* uniforms, const int32_t* parents, const int32_t* cu,
                                       const int32_t* slots, int32_t rows, int32_t max_new, float temperature,
                                       const float* temperatures, int32_t* accepted, int32_t* path, int32_t* out_tokens,
                                       int dtype, void* ws, int64_t ws_bytes, void* stream) {
  if (const int rc = check_sizes(tokens, rows, vocab, max_new, dtype)) return rc;
  if (!cu && tokens != (int64_t)rows * max_new)
    return fail(BSG_ERR_ARG, "without cu, tokens=%lld must be rows x max_new = %lld", (long long)tokens, (long long)rows * max_new);
  if (draft_logits && parents) return fail(BSG_ERR_UNSUPPORTED, "draft_logits go with chains: parents must be NULL");
  if (!temperatures && !(temperature >= 0.f && temperature < __builtin_inff()))
    return fail(BSG_ERR_ARG, "temperature=%g", temperature);
  if (rows == 0) return BSG_OK;
  if (!accepted || (max_new > 0 && (!path || !out_tokens)))
    return fail(BSG_ERR_ARG, "null pointer (accepted=%p path=%p out_tokens=%p)", (void*)accepted, (void*)path, (void*)out_tokens);
  if (tokens > 0 && (!logits || !token_ids || !uniforms))
    return fail(BSG_ERR_ARG, "null pointer (logits=%p token_ids=%p uniforms=%p)", logits, (const void*)token_ids, (const void*)uniforms);
  const int drafts = draft_logits != nullptr;
  const unsigned size = dtype == BSG_F32 ? 4 : 2;
  if (!is_aligned(logits, size) || !is_aligned(draft_logits, size))
    return fail(BSG_ERR_ALIGN, "logits must be aligned to their type");
  const Layout l = layout_of(tokens, rows, vocab, drafts);
  if (!ws || ws_bytes < l.bytes)
    return fail(BSG_ERR_WORKSPACE, "workspace of %lld bytes, %lld needed", (long long)ws_bytes, (long long)l.bytes);
  if (!is_aligned(ws, 16)) return fail(BSG_ERR_ALIGN, "workspace must be 16-byte aligned");
  VerifyParams p;
  p.x[0] = logits, p.x[1] = draft_logits;
  p.stride[0] = logits_stride, p.stride[1] = draft_stride;
  p.vocab = vocab, p.tokens = tokens;
  p.ids = token_ids, p.uniforms = uniforms, p.parents = parents, p.cu = cu, p.slots = slots;
  p.temperatures = temperatures, p.temperature = temperature;
  p.rows = rows, p.max_new = max_new, p.drafts = drafts;
  p.pieces = (int32_t)l.pieces, p.groups = (int32_t)ceil_div(l.pieces, kWaves);
  p.accepted = accepted, p.path = path, p.out = out_tokens;
  p.counters = (uint32_t*)ws;
  p.stats = (Piece*)((uint8_t*)ws + l.stats);
  p.last = (Piece*)((uint8_t*)ws + l.last);
  const hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case BSG_F16: launch<_Float16>(p, st); break;
    case BSG_BF16: launch<__bf16>(p, st); break;
    default: launch<float>(p, st); break;
  }
  return launch_status("bsg_verify_drafts");
}
