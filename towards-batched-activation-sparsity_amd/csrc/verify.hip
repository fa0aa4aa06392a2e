// verify.hip — which drafted tokens a target model accepts, and the token that follows them (include/bsgdraft.h).
//
// Answers are whole numbers next to borders: a number u against a ratio of probabilities, and the first running sum past
// u of the whole.  So weights w = 2^((x - m) k), k = log2(e) / temperature, and their sums are 64-bit.  2^t is
// 2^n times the Taylor polynomial of e^(f ln 2), t = n + f, |f| <= 1/2, to the 12th power (relative error
// (ln 2 / 2)^13 / 13! = 1.7e-16).
//
// First launch: a wave has kPiece consecutive logits of one node's row in registers and leaves their maximum and
// the sum of their weights against it (or, greedy, where the first maximum is).  The last work-group of a sequence to arrive
// has all of them: it walks the tree (a node in each lane; nodes in order, each asked if its parent is the last accepted
// one) and draws the new token from the last row, whose pieces' sums it already has: the piece by them, the token by reading
// that piece again.  Second launch, where drafts come with probabilities: the sums of max(p - q, 0) over the pieces of
// a row whose child was rejected, and the draw from those.

#include "bsgdraft.h"
#include "draft_tree.hpp"

using namespace bsgk;

namespace {

constexpr int kPiece = 2048;  // logits of a wave
constexpr int kWaves = 4;     // of a work-group
constexpr int kMostPieces = 512;  // of a row
constexpr double kLog2e = 1.4426950408889634;

struct Piece {  // of a row
  double sum;   // of its weights; NaN: a logit is NaN or +inf
  float top;
  int32_t at;   // of the first maximum
};
struct Verdict {  // what the first launch leaves the second
  double total[2];  // of p's and q's row, against the maxima
  float top[2];
  int32_t node, count, residual, pad;  // residual: the row whose max(p - q, 0) is drawn from is node's
};

struct VerifyParams {
  const void* x[2];  // the target's logits, the drafts'
  int64_t stride[2];
  int64_t vocab, tokens;
  const int32_t* ids;
  const float* uniforms;
  const int32_t* parents;
  const int32_t* cu;
  const float* temperatures;
  float temperature;
  int32_t rows, max_new, pieces, groups, drafts;  // pieces of a row, work-groups of a row
  int32_t* accepted;
  int32_t* path;
  int32_t* out;
  uint32_t* counters;  // [rows]: the first launch's, then the second's
  Verdict* verdicts;   // [rows]
  Piece* stats;        // [tokens][1 + drafts][pieces]
  double* left;        // [rows][pieces]
};

// 2^t for t <= 0, and 0 far below.
__device__ __forceinline__ double exp2_64(double t) {
  t = t < -1100.0 ? -1100.0 : t;
  const double n = __builtin_rint(t), f = t - n;
  // (ln 2)^i / i!
  double y = 2.5678435993488206e-11;
  y = __builtin_fma(y, f, 4.4455382718708115e-10);
  y = __builtin_fma(y, f, 7.0549116208011234e-09);
  y = __builtin_fma(y, f, 1.0178086009239699e-07);
  y = __builtin_fma(y, f, 1.3215486790144309e-06);
  y = __builtin_fma(y, f, 1.5252733804059841e-05);
  y = __builtin_fma(y, f, 0.00015403530393381609);
  y = __builtin_fma(y, f, 0.0013333558146428443);
  y = __builtin_fma(y, f, 0.0096181291076284772);
  y = __builtin_fma(y, f, 0.055504108664821580);
  y = __builtin_fma(y, f, 0.24022650695910071);
  y = __builtin_fma(y, f, 0.69314718055994531);
  y = __builtin_fma(y, f, 1.0);
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

// A wave's piece of a row: vector v of lane l holds the logits piece * kPiece + (64 v + l) PER .. of the row, -inf past its
// end.  Rows that 16 bytes do not divide come number by number.
template <typename T>
struct PieceOf {
  static constexpr int PER = Logit<T>::PER, VECTORS = kPiece / 64 / PER;
  u32x4 v[VECTORS];
  __device__ __forceinline__ void load(const void* x, int64_t row_at, int64_t vocab, int piece, int lane) {
    const T* const row = (const T*)x + row_at;
    const bool wide = ((uintptr_t)row & 15) == 0;
#pragma unroll
    for (int k = 0; k < VECTORS; ++k) {
      const int64_t at = (int64_t)piece * kPiece + (64 * k + lane) * PER;
      if (wide && at + PER <= vocab) {
        v[k] = *(const u32x4*)(row + at);
      } else {
        typedef T vec __attribute__((ext_vector_type(PER)));
        vec w;
#pragma unroll
        for (int e = 0; e < PER; ++e) w[e] = at + e < vocab ? row[at + e] : (T)-__builtin_inff();
        v[k] = __builtin_bit_cast(u32x4, w);
      }
    }
  }
  __device__ __forceinline__ float get(int k, int e) const { return Logit<T>::of(v[k], e); }
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

// The weight of a logit against a maximum; 0 for -inf.
__device__ __forceinline__ double weight(float x, float top, double k) {
  return x == -__builtin_inff() ? 0.0 : exp2_64(((double)x - (double)top) * k);
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
  const bool fine = t.from >= 0 && t.from < to && to <= p.tokens;
  t.count = !fine ? 0 : to - t.from < p.max_new ? (int)(to - t.from) : p.max_new;
  t.parent = load_parent(p.parents, t.from, t.count, lane);
  return t;
}

__device__ __forceinline__ const Piece* piece_at(const VerifyParams& p, int64_t token, int which) {
  return p.stats + (token * (1 + p.drafts) + which) * p.pieces;
}
__device__ __forceinline__ Piece load_piece(const Piece* at) {
  Piece v;
  v.sum = __builtin_bit_cast(double, hand_load((const uint64_t*)at));
  const uint64_t b = hand_load((const uint64_t*)at + 1);
  v.top = as_float((uint32_t)b), v.at = (int32_t)(b >> 32);
  return v;
}

// A row's maximum, the sum of its weights against it and where the first maximum is, from its pieces: a wave's work.
struct Row {
  double total;
  float top;
  int32_t at;
};
__device__ __forceinline__ Row row_of(const Piece* pieces, int n, double k, int lane) {
  Row r = {0.0, -__builtin_inff(), 0x7fffffff};
  for (int c0 = 0; c0 < n; c0 += 64) {
    Piece v = {0.0, -__builtin_inff(), 0x7fffffff};
    if (c0 + lane < n) v = load_piece(pieces + c0 + lane);
    const float top = fmaxf(r.top, wave_max<32>(v.top));
    const int at = wave_min<32>(v.top == top ? v.at : 0x7fffffff);
    if (top > r.top || c0 == 0) r.at = at;
    const double sum = wave_sum<32>(v.sum == v.sum ? v.sum * weight(v.top, top, k) : v.sum);
    r.total = (r.top == -__builtin_inff() ? r.total : r.total * weight(r.top, top, k)) + sum;
    r.top = top;
  }
  return r;
}

__device__ __forceinline__ double read_lane(double v, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)b, lane), hi = __builtin_amdgcn_readlane((int)(b >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// The first piece of a row whose running sum passes `goal`, the last one of any weight if none does; `before` gets the
// sum before it.
template <typename Sum>
__device__ __forceinline__ int pick_piece(int n, double goal, int lane, double* before, const Sum& sum) {
  double run = 0.0, last_before = 0.0;
  int last = -1;
  for (int c0 = 0; c0 < n; c0 += 64) {
    const double v = c0 + lane < n ? sum(c0 + lane) : 0.0;
    const double upto = run + wave_scan(v, lane);
    const uint64_t past = __ballot(upto > goal && v > 0.0), some = __ballot(v > 0.0);
    const int at = past ? __builtin_ctzll(past) : some ? 63 - __builtin_clzll(some) : -1;
    if (at >= 0) {
      last = c0 + at;
      last_before = read_lane(upto - v, at);
      if (past) break;
    }
    run = read_lane(upto, 63);
  }
  *before = last_before;
  return last;
}

// The first token of a piece whose running sum, from `before` on, passes `goal`; the last one of any weight if none does.
template <typename T, typename Weight>
__device__ __forceinline__ int pick_token(int piece, double before, double goal, int lane, const Weight& weight_of) {
  constexpr int PER = PieceOf<T>::PER, VECTORS = PieceOf<T>::VECTORS;
  int found = -1, last = -1;
#pragma unroll
  for (int k = 0; k < VECTORS; ++k) {
    if (found >= 0) continue;
    double v[PER], sum = 0.0;
#pragma unroll
    for (int e = 0; e < PER; ++e) v[e] = weight_of(k, e), sum += v[e];
    const double upto = before + wave_scan(sum, lane);
    double run = upto - sum;
    int hit = -1, any = -1;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      run += v[e];
      if (v[e] > 0.0) {
        any = e;
        if (hit < 0 && run > goal) hit = e;
      }
    }
    // what passes by the scan's sum passes here, where the lane's own may be short of it by a last bit
    if (hit < 0 && any >= 0 && upto > goal) hit = any;
    const uint64_t past = __ballot(hit >= 0), some = __ballot(any >= 0);
    const int base = piece * kPiece + 64 * k * PER;
    if (past) {
      const int at = __builtin_ctzll(past);
      found = base + at * PER + __builtin_amdgcn_readlane(hit, at);
    }
    if (some) {
      const int at = 63 - __builtin_clzll(some);
      last = base + at * PER + __builtin_amdgcn_readlane(any, at);
    }
    before = read_lane(upto, 63);
  }
  return found >= 0 ? found : last;
}

// The sequence's answer: the accepted nodes (a bit for each), the new token.  A wave's work.
__device__ __forceinline__ void answer(const VerifyParams& p, int row, const Tree& t, uint64_t taken, int token, int lane) {
  const int count = __builtin_popcountll(taken);
  int32_t* const path = p.path + (int64_t)row * p.max_new;
  int32_t* const out = p.out + (int64_t)row * p.max_new;
  const int place = __builtin_popcountll(taken & ((1ull << lane) - 1));
  const bool mine = taken >> lane & 1;
  if (mine) path[place] = lane;
  if (mine && place > 0) out[place - 1] = p.ids[t.from + lane];
  if (lane == 0 && count > 0) out[count - 1] = token;
  for (int i = count + lane; i < p.max_new; i += 64) path[i] = -1, out[i] = -1;
  if (lane == 0) p.accepted[row] = count;
}

template <typename T>
__global__ __launch_bounds__(64 * kWaves) void bsg_verify_rows_kernel(VerifyParams p) {
  __shared__ double s_total[2][BSG_TREE_NODES];
  __shared__ float s_top[2][BSG_TREE_NODES];
  __shared__ int32_t s_at[BSG_TREE_NODES];
  __shared__ uint32_t s_last;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int which = blockIdx.x / p.groups, group = blockIdx.x - which * p.groups;
  const int node = blockIdx.y, row = blockIdx.z;
  const Tree t = tree_of(p, row, lane);
  if (node >= t.count) {
    if (t.count == 0 && node == 0 && blockIdx.x == 0 && wave == 0) answer(p, row, t, 0, -1, lane);
    return;
  }
  const bool greedy = !(t.temperature > 0.f);
  const double k = greedy ? 1.0 : kLog2e / (double)t.temperature;
  const int piece = group * kWaves + wave;
  if (piece < p.pieces && !(greedy && which)) {
    PieceOf<T> x;
    x.load(p.x[which], (t.from + node) * p.stride[which], p.vocab, piece, lane);
    float top = -__builtin_inff();
    bool bad = false;
#pragma unroll
    for (int v = 0; v < PieceOf<T>::VECTORS; ++v)
#pragma unroll
      for (int e = 0; e < PieceOf<T>::PER; ++e) {
        const float y = x.get(v, e);
        top = fmaxf(top, y);
        bad = bad || !(y < __builtin_inff());
      }
    top = wave_max<32>(top);
    Piece mine = {0.0, top, 0x7fffffff};
    if (greedy) {
#pragma unroll
      for (int v = PieceOf<T>::VECTORS - 1; v >= 0; --v)
#pragma unroll
        for (int e = PieceOf<T>::PER - 1; e >= 0; --e)
          if (x.get(v, e) == top) mine.at = piece * kPiece + (64 * v + lane) * PieceOf<T>::PER + e;
      mine.at = wave_min<32>(mine.at);
    } else if (top > -__builtin_inff()) {
#pragma unroll
      for (int v = 0; v < PieceOf<T>::VECTORS; ++v)
#pragma unroll
        for (int e = 0; e < PieceOf<T>::PER; ++e) mine.sum += exp2_64(((double)x.get(v, e) - (double)top) * k);
      mine.sum = wave_sum<32>(mine.sum);
    }
    if (__any(bad)) mine.sum = __builtin_nan("");
    if (lane == 0) {
      uint64_t* const at = (uint64_t*)(piece_at(p, t.from + node, which) + piece);
      hand_store(at, __builtin_bit_cast(uint64_t, mine.sum));
      hand_store(at + 1, (uint64_t)(uint32_t)mine.at << 32 | __builtin_bit_cast(uint32_t, mine.top));
    }
  }
  hand_publish();
  __syncthreads();
  const uint32_t arrivals = (uint32_t)t.count * p.groups * (1 + p.drafts);
  if (threadIdx.x == 0) s_last = hand_arrive(p.counters + row) == arrivals - 1;
  __syncthreads();
  if (!s_last) return;
  if (threadIdx.x == 0) hand_reset(p.counters + row);

  // this work-group has the sequence: its rows' maxima and sums
  const bool drafts = p.drafts != 0 && !greedy;
  for (int r = wave; r < (drafts ? 2 * t.count : t.count); r += kWaves) {
    const int w = r >= t.count, i = w ? r - t.count : r;
    const Row v = row_of(piece_at(p, t.from + i, w), p.pieces, k, lane);
    if (lane == 0) {
      s_total[w][i] = v.total, s_top[w][i] = v.top;
      if (!w) s_at[i] = v.at;
    }
  }
  __syncthreads();
  if (wave != 0) return;

  // node `lane`: its token's weight in its parent's row, and in the drafts'
  const int up = t.parent < 0 ? 0 : t.parent;
  const int id = lane < t.count ? p.ids[t.from + lane] : -1;
  const double u = lane < t.count ? (double)p.uniforms[t.from + lane] : 0.0;
  const bool child = t.parent >= 0, known = child && id >= 0 && id < p.vocab;
  double mine = 0.0, theirs = 0.0;
  if (known && !greedy) {
    mine = weight(Logit<T>::one(p.x[0], (t.from + up) * p.stride[0] + id), s_top[0][up], k);
    if (drafts) {
      mine /= s_total[0][up];
      theirs = weight(Logit<T>::one(p.x[1], (t.from + up) * p.stride[1] + id), s_top[1][up], k) / s_total[1][up];
    }
  }
  int at = 0;
  uint64_t taken = 1, refused = 0;  // refused: the rejected children of `at`, of each token one
  double out = 0.0;                 // their weights
  for (uint64_t left = ~1ull;;) {
    const uint64_t asked = left & __ballot(child && t.parent == at);
    if (!asked) break;
    const int j = __builtin_ctzll(asked);
    left = j == 63 ? 0 : left & ~0ull << (j + 1);
    const bool same = (refused & __ballot(id == __builtin_amdgcn_readlane(id, j))) != 0;  // has no weight left
    const bool ok = greedy ? id == s_at[at] && s_total[0][at] == s_total[0][at] : drafts ? u * theirs < mine : u * (s_total[0][at] - out) < mine;
    if (!same && (__ballot(ok && known) >> j & 1) != 0) {
      at = j, taken |= 1ull << j, refused = 0, out = 0.0;
    } else if (!same) {
      refused |= 1ull << j, out += read_lane(mine, j);
    }
  }

  // the new token
  const double total = s_total[0][at];
  const float top = s_top[0][at];
  const bool residual = drafts && refused != 0;
  int token = -1;
  if (greedy) {
    if (total == total && top > -__builtin_inff()) token = s_at[at];
  } else if (total > 0.0 && !residual) {
    // what is left of the row: the rejected tokens' weights go out of their pieces
    double rest = total - out;
    if (!(rest > 0.0)) rest = total, refused = 0;
    const double goal = read_lane(u, 0) * rest;
    const Piece* const pieces = piece_at(p, t.from + at, 0);
    double before;
    const int c = pick_piece(p.pieces, goal, lane, &before, [&](int i) {
      const Piece v = load_piece(pieces + i);
      double sum = v.sum * weight(v.top, top, k);
      for (uint64_t m = refused; m; m &= m - 1) {
        const int j = __builtin_ctzll(m), gone = __builtin_amdgcn_readlane(id, j);
        if (gone >= 0 && gone / kPiece == i) sum -= read_lane(mine, j);
      }
      return sum;
    });
    if (c >= 0) {
      PieceOf<T> x;
      x.load(p.x[0], (t.from + at) * p.stride[0], p.vocab, c, lane);
      uint32_t gone = 0;  // of the lane's numbers, as bits
      for (uint64_t m = refused; m; m &= m - 1) {
        const int off = __builtin_amdgcn_readlane(id, __builtin_ctzll(m)) - c * kPiece;
        if (off >= 0 && off < kPiece && off / PieceOf<T>::PER % 64 == lane)
          gone |= 1u << (off / PieceOf<T>::PER / 64 * PieceOf<T>::PER + off % PieceOf<T>::PER);
      }
      token = pick_token<T>(c, before, goal, lane, [&](int v, int e) {
        return gone >> (v * PieceOf<T>::PER + e) & 1 ? 0.0 : weight(x.get(v, e), top, k);
      });
    }
  }
  answer(p, row, t, taken, token, lane);
  if (p.drafts && lane == 0) {
    Verdict v;
    v.total[0] = total, v.total[1] = s_total[1][at];
    v.top[0] = top, v.top[1] = s_top[1][at];
    v.node = at, v.count = __builtin_popcountll(taken), v.residual = residual && total > 0.0, v.pad = 0;
    p.verdicts[row] = v;
  }
}

// The new token of the sequences whose last row's child was rejected, from max(p - q, 0); from p where nothing is left.
template <typename T>
__global__ __launch_bounds__(64 * kWaves) void bsg_verify_residual_kernel(VerifyParams p) {
  __shared__ uint32_t s_last;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = blockIdx.y;
  const Tree t = tree_of(p, row, lane);
  if (t.count == 0 || !(t.temperature > 0.f)) return;
  const Verdict v = p.verdicts[row];
  if (!v.residual) return;
  const double k = kLog2e / (double)t.temperature;
  const double by[2] = {1.0 / v.total[0], 1.0 / v.total[1]};
  const int64_t at[2] = {(t.from + v.node) * p.stride[0], (t.from + v.node) * p.stride[1]};
  double* const left = p.left + (int64_t)row * p.pieces;
  const auto of = [&](const PieceOf<T>& x, const PieceOf<T>& y, int i, int e) {
    const double d = weight(x.get(i, e), v.top[0], k) * by[0] - weight(y.get(i, e), v.top[1], k) * by[1];
    return d > 0.0 ? d : 0.0;
  };
  PieceOf<T> x, y;
  const int piece = blockIdx.x * kWaves + wave;
  if (piece < p.pieces) {
    x.load(p.x[0], at[0], p.vocab, piece, lane);
    y.load(p.x[1], at[1], p.vocab, piece, lane);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < PieceOf<T>::VECTORS; ++i)
#pragma unroll
      for (int e = 0; e < PieceOf<T>::PER; ++e) sum += of(x, y, i, e);
    sum = wave_sum<32>(sum);
    if (lane == 0) hand_store((uint64_t*)left + piece, __builtin_bit_cast(uint64_t, sum));
  }
  hand_publish();
  __syncthreads();
  if (threadIdx.x == 0) s_last = hand_arrive(p.counters + row) == (uint32_t)(p.groups - 1);
  __syncthreads();
  if (!s_last) return;
  if (threadIdx.x == 0) hand_reset(p.counters + row);
  if (wave != 0) return;

  double total = 0.0;
  for (int c = lane; c < p.pieces; c += 64) total += __builtin_bit_cast(double, hand_load((const uint64_t*)left + c));
  total = wave_sum<32>(total);
  const bool some = total > 0.0;
  const Piece* const pieces = piece_at(p, t.from + v.node, 0);
  const double goal = (double)p.uniforms[t.from] * (some ? total : v.total[0]);
  double before;
  const int c = pick_piece(p.pieces, goal, lane, &before, [&](int i) {
    if (some) return __builtin_bit_cast(double, hand_load((const uint64_t*)left + i));
    const Piece w = load_piece(pieces + i);
    return w.sum * weight(w.top, v.top[0], k);
  });
  int token = -1;
  if (c >= 0) {
    x.load(p.x[0], at[0], p.vocab, c, lane);
    y.load(p.x[1], at[1], p.vocab, c, lane);
    token = pick_token<T>(c, before, goal, lane, [&](int i, int e) {
      return some ? of(x, y, i, e) : weight(x.get(i, e), v.top[0], k);
    });
  }
  if (lane == 0) p.out[(int64_t)row * p.max_new + v.count - 1] = token;
}

struct Layout {
  int64_t pieces, verdicts, stats, left, bytes;  // of a row; where they lie in the workspace
};
Layout layout_of(int64_t tokens, int32_t rows, int64_t vocab, int32_t drafts) {
  Layout l;
  l.pieces = ceil_div(vocab, kPiece);
  l.verdicts = BSG_KV_COUNTER_BYTES;
  l.stats = l.verdicts + ceil_div((drafts ? rows : 0) * (int64_t)sizeof(Verdict), 256) * 256;
  l.left = l.stats + tokens * (1 + drafts) * l.pieces * (int64_t)sizeof(Piece);
  l.bytes = l.left + (drafts ? rows * l.pieces * 8 : 0);
  return l;
}

int check_sizes(int64_t tokens, int32_t rows, int64_t vocab, int32_t max_new, int dtype) {
  if (dtype != BSG_F16 && dtype != BSG_BF16 && dtype != BSG_F32) return fail(BSG_ERR_DTYPE, "dtype=%d (0=fp16, 1=bf16, 2=fp32)", dtype);
  if (tokens < 0 || rows < 0 || vocab < 1 || max_new < 0 || tokens > 0x7fffffff)
    return fail(BSG_ERR_ARG, "tokens=%lld rows=%d vocab=%lld max_new=%d", (long long)tokens, rows, (long long)vocab, max_new);
  if (max_new > BSG_TREE_NODES) return fail(BSG_ERR_UNSUPPORTED, "%d nodes in a tree (at most %d)", max_new, BSG_TREE_NODES);
  if (vocab > (int64_t)kMostPieces * kPiece) return fail(BSG_ERR_UNSUPPORTED, "vocab=%lld (at most %d)", (long long)vocab, kMostPieces * kPiece);
  if (rows > BSG_KV_COUNTER_BYTES / 4) return fail(BSG_ERR_UNSUPPORTED, "%d sequences (at most %d)", rows, BSG_KV_COUNTER_BYTES / 4);
  return BSG_OK;
}

template <typename T>
void launch(const VerifyParams& p, hipStream_t st) {
  const dim3 grid((unsigned)(p.groups * (1 + p.drafts)), (unsigned)p.max_new, (unsigned)p.rows);
  hipLaunchKernelGGL((bsg_verify_rows_kernel<T>), grid, dim3(64 * kWaves), 0, st, p);
  if (p.drafts)
    hipLaunchKernelGGL((bsg_verify_residual_kernel<T>), dim3((unsigned)p.groups, (unsigned)p.rows), dim3(64 * kWaves), 0, st, p);
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
  if (const int rc = check_sizes(tokens, rows, vocab, max_new, dtype)) return rc;
  if (!cu && tokens != (int64_t)rows * max_new)
    return fail(BSG_ERR_ARG, "without cu, tokens=%lld must be rows x max_new = %lld", (long long)tokens, (long long)rows * max_new);
  if (draft_logits && parents) return fail(BSG_ERR_UNSUPPORTED, "draft_logits go with chains: parents must be NULL");
  if (!temperatures && !(temperature >= 0.f && temperature < __builtin_inff()))
    return fail(BSG_ERR_ARG, "temperature=%g", temperature);
  if (rows == 0 || max_new == 0) return BSG_OK;
  if (!accepted || !path || !out_tokens)
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
  p.ids = token_ids, p.uniforms = uniforms, p.parents = parents, p.cu = cu;
  p.temperatures = temperatures, p.temperature = temperature;
  p.rows = rows, p.max_new = max_new, p.drafts = drafts;
  p.pieces = (int32_t)l.pieces, p.groups = (int32_t)ceil_div(l.pieces, kWaves);
  p.accepted = accepted, p.path = path, p.out = out_tokens;
  p.counters = (uint32_t*)ws;
  p.verdicts = (Verdict*)((uint8_t*)ws + l.verdicts);
  p.stats = (Piece*)((uint8_t*)ws + l.stats);
  p.left = (double*)((uint8_t*)ws + l.left);
  const hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case BSG_F16: launch<_Float16>(p, st); break;
    case BSG_BF16: launch<__bf16>(p, st); break;
    default: launch<float>(p, st); break;
  }
  return launch_status("bsg_verify_drafts");
}
