// logprobs.hip — log probabilities of given tokens, entropies and the likeliest alternatives of rows of
// logits, in one pass over them (include/bsgserve.h).
//
// With M the running maximum of a row, l = sum 2^d and t = sum 2^d d over d = (x - M) log2(e):
//   lse = M + ln l,  logprob = (x_token - M) - ln l,  entropy = ln 2 (log2 l - t / l).
// The alternatives are found beside it.  A logit's key is its order among fp32 numbers (upper half) and
// its id's complement (lower half), so that keys are distinct and (logit desc, id asc) is key desc.  The k
// best keys so far wait in LDS; a tile of logits in registers adds to them what passes a threshold
// that at least k keys reach: the worst of the k, or on the first tile the k-th largest of some
// wave's 64 lane maxima.

#include "serve.hpp"

using namespace bsgk;

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kVectors = 4;     // 16-byte vectors of a thread and tile
constexpr int kList = 1024;     // candidates of one round; more of them take the search by bits
constexpr int kMaxK = BSG_LOGPROBS_MAX_K;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
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
  int32_t k, splits;
};

template <typename T>
struct Logit;
template <>
struct Logit<_Float16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float at(const u32x4& v, int i) {
    return i & 1 ? high_half<_Float16>(v[i >> 1]) : low_half<_Float16>(v[i >> 1]);
  }
};
template <>
struct Logit<__bf16> {
  static constexpr int N = 8;
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

struct Sums {
  float m, l, t;
};
__device__ __forceinline__ Sums join(Sums a, Sums b) {
  const float m = fmaxf(a.m, b.m);
  if (m == -__builtin_inff()) return Sums{m, a.l + b.l, a.t + b.t};
  const float da = fmaxf((a.m - m) * kLog2e, kFloor), db = fmaxf((b.m - m) * kLog2e, kFloor);
  const float fa = __builtin_amdgcn_exp2f(da), fb = __builtin_amdgcn_exp2f(db);
  return Sums{m, a.l * fa + b.l * fb, fa * (a.t + a.l * da) + fb * (b.t + b.l * db)};
}

// The k-th largest (from 1) of the wave's 64 values: a bitonic sort of one value per lane, largest first.
__device__ __forceinline__ uint32_t wave_kth(uint32_t v, int k) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int n = 2; n <= 64; n <<= 1)
#pragma unroll
    for (int j = n >> 1; j > 0; j >>= 1) {
      const uint32_t o = __shfl_xor(v, j);
      const bool larger = ((lane & j) == 0) == ((lane & n) == 0 || n == 64);
      v = larger ? (v > o ? v : o) : (v < o ? v : o);
    }
  return __builtin_amdgcn_readlane(v, k - 1);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void bsg_token_logprobs_kernel(ScoreParams p) {
  typedef Logit<T> L;
  constexpr int N = L::N;
  __shared__ uint64_t s_list[kList + kMaxK];
  __shared__ uint64_t s_top[kMaxK];
  __shared__ uint32_t s_tau[kWaves];
  __shared__ Sums s_sum[kWaves];
  __shared__ uint32_t s_counts[2], s_last;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.y;
  const T* const x = (const T*)p.x + row * p.stride;
  // 16-byte vectors from the granule in which the row begins: its element i is at i + skip
  const int skip = (int)(((uintptr_t)x & 15u) / sizeof(T));
  const int64_t vectors = (p.vocab + skip + N - 1) / N;
  const int64_t v_begin = (int64_t)blockIdx.x * p.split_vectors;
  const int64_t v_end = v_begin + p.split_vectors < vectors ? v_begin + p.split_vectors : vectors;
  const int k = p.k;

  Sums sum = {-__builtin_inff(), 0.f, 0.f};
  int have = 0;  // keys in s_top, sorted
  if (tid < 2) s_counts[tid] = 0;
  __syncthreads();
  int turn = 0;
  for (int64_t v0 = v_begin; v0 < v_end; v0 += kThreads * kVectors) {
    // counters by turns: threads that go on with nothing found may count again while others still read
    uint32_t& s_count = s_counts[turn];
    turn ^= 1;
    u32x4 raw[kVectors];
    uint32_t valid[kVectors];  // one bit per element
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      const int64_t v = v0 + i * kThreads + tid;
      const int64_t e = v * N - skip;
      valid[i] = 0;
      raw[i] = u32x4{0u, 0u, 0u, 0u};
      if (v < v_end) {
        if (e >= 0 && e + N <= p.vocab) {
          raw[i] = __builtin_nontemporal_load((const u32x4*)(x + e));
          valid[i] = (1u << N) - 1u;
        } else {
#pragma unroll
          for (int j = 0; j < N; ++j)
            if (e + j >= 0 && e + j < p.vocab) {
              valid[i] |= 1u << j;
              if constexpr (sizeof(T) == 4)
                raw[i][j] = ((const uint32_t*)x)[e + j];
              else
                raw[i][j >> 1] |= (uint32_t)((const uint16_t*)x)[e + j] << (16 * (j & 1));
            }
        }
      }
    }
    const auto logit = [&](int i, int j) { return valid[i] >> j & 1u ? L::at(raw[i], j) : -__builtin_inff(); };
    const auto order = [&](int i, int j) { return valid[i] >> j & 1u ? order_of(L::at(raw[i], j)) : 0u; };

    float m = sum.m;
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) m = fmaxf(m, logit(i, j));
    const float base = m == -__builtin_inff() ? 0.f : m;
    float l = 0.f, t = 0.f;
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float d = (logit(i, j) - base) * kLog2e;
        const float e = __builtin_amdgcn_exp2f(d);
        l += e;
        t += e * fmaxf(d, kFloor);
      }
    sum = join(sum, Sums{m, l, t});

    if (k == 0) continue;
    uint32_t tau;
    if (have == k) {
      tau = (uint32_t)(s_top[k - 1] >> 32);
    } else {
      uint32_t best = 0;
#pragma unroll
      for (int i = 0; i < kVectors; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const uint32_t o = order(i, j);
          best = best > o ? best : o;
        }
      tau = wave_kth(best, k);
      if (lane == 0) s_tau[wave] = tau;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWaves; ++w) tau = tau > s_tau[w] ? tau : s_tau[w];
    }
    const uint64_t worst = have == k ? s_top[k - 1] : 0;
    // positions are taken by an atomic; the ranks below make their order irrelevant
    int mine = 0;
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const uint32_t o = order(i, j);
        mine += o != 0 && o >= tau;
      }
    if (mine > 0) {
      uint32_t at = atomicAdd(&s_count, (uint32_t)mine);
#pragma unroll
      for (int i = 0; i < kVectors; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const uint32_t o = order(i, j);
          if (o != 0 && o >= tau) {
            if (at < kList) s_list[at] = key_of(o, (uint32_t)((v0 + i * kThreads + tid) * N - skip + j));
            ++at;
          }
        }
    }
    __syncthreads();
    int n = (int)s_count;
    if (n == 0) continue;
    if (n > kList) {
      // Too many equal or ascending logits for the list: the k-th largest key, one bit at a time.
      uint64_t kth = 0;
      for (int bit = 63; bit >= 0; --bit) {
        const uint64_t probe = kth | (uint64_t)1 << bit;
        int c = 0;
#pragma unroll
        for (int i = 0; i < kVectors; ++i)
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const uint32_t o = order(i, j);
            c += o != 0 && key_of(o, (uint32_t)((v0 + i * kThreads + tid) * N - skip + j)) >= probe;
          }
        __syncthreads();
        if (tid == 0) s_count = 0;
        __syncthreads();
        if (c > 0) atomicAdd(&s_count, (uint32_t)c);
        __syncthreads();
        if ((int)s_count >= k) kth = probe;
      }
      __syncthreads();
      if (tid == 0) s_count = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kVectors; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const uint32_t o = order(i, j);
          const uint64_t key = key_of(o, (uint32_t)((v0 + i * kThreads + tid) * N - skip + j));
          if (o != 0 && key >= kth) s_list[atomicAdd(&s_count, 1u)] = key;
        }
      __syncthreads();
      n = (int)s_count;
    }
    if (tid < have) s_list[n + tid] = s_top[tid];
    __syncthreads();
    const int all = n + have;
    for (int e = tid; e < all; e += kThreads) {
      const uint64_t key = s_list[e];
      if (key < worst) continue;
      int rank = 0;
      for (int i = 0; i < all; ++i) rank += s_list[i] > key;
      if (rank < k) s_top[rank] = key;
    }
    have = all < k ? all : k;
    if (tid == 0) s_count = 0;
    __syncthreads();
  }

#pragma unroll
  for (int d = 1; d < 64; d <<= 1)
    sum = join(sum, Sums{__shfl_xor(sum.m, d), __shfl_xor(sum.l, d), __shfl_xor(sum.t, d)});
  if (lane == 0) s_sum[wave] = sum;
  __syncthreads();
  sum = s_sum[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) sum = join(sum, s_sum[w]);

  if (p.splits > 1) {
    const int64_t at = row * p.splits + blockIdx.x;
    if (tid < k) hand_store(p.keys + at * k + tid, tid < have ? s_top[tid] : (uint64_t)0);
    if (tid == 0) hand_store(p.sums + at * 4, sum.m), hand_store(p.sums + at * 4 + 1, sum.l), hand_store(p.sums + at * 4 + 2, sum.t);
    hand_publish();
    __syncthreads();
    if (tid == 0) s_last = hand_arrive(p.counters + row) == (uint32_t)(p.splits - 1);
    __syncthreads();
    if (!s_last) return;
    if (tid == 0) hand_reset(p.counters + row);
    const int64_t first = row * p.splits;
    sum = Sums{-__builtin_inff(), 0.f, 0.f};
    for (int s = 0; s < p.splits; ++s)
      sum = join(sum, Sums{hand_load(p.sums + (first + s) * 4), hand_load(p.sums + (first + s) * 4 + 1),
                           hand_load(p.sums + (first + s) * 4 + 2)});
    const int all = p.splits * k;  // at most kList
    if (tid < all) s_list[tid] = hand_load(p.keys + first * k + tid);
    __syncthreads();
    if (tid < all && s_list[tid] != 0) {
      const uint64_t key = s_list[tid];
      int rank = 0;
      for (int i = 0; i < all; ++i) rank += s_list[i] > key;
      if (rank < k) s_top[rank] = key;
    }
    __syncthreads();
  }

  // a NaN is in l even where it was never the maximum; nothing but -inf has l = 0
  const float log_l = __builtin_amdgcn_logf(sum.l);
  const float top = sum.m == -__builtin_inff() ? 0.f : sum.m;
  const auto logprob = [&](float v) { return sum.l == 0.f ? v : (v - top) - log_l * kLn2; };
  if (tid < k) {
    const uint64_t key = s_top[tid];
    p.top_ids[row * k + tid] = (int32_t)~(uint32_t)key;
    p.top_logprobs[row * k + tid] = logprob(from_order((uint32_t)(key >> 32)));
  }
  if (tid == 0) {
    const int32_t token = p.tokens[row];
    p.logprob[row] = token >= 0 && token < p.vocab ? logprob((float)x[token]) : __builtin_nanf("");
    p.entropy[row] = sum.l == 0.f ? 0.f : kLn2 * (log_l - sum.t / sum.l);
  }
}

struct Shape {
  int32_t splits;
  int64_t split_vectors;
};

// Rows alone fill the machine from two work-groups per compute unit on; fewer rows are split, down to one
// vector per thread, and to what one list of alternatives holds.
Shape shape_of(int64_t rows, int64_t vocab, int32_t k, int per_vector, int32_t cus) {
  const int64_t vectors = ceil_div(vocab, per_vector) + 1;  // a row may begin inside a vector
  int64_t want = ceil_div(2 * (int64_t)cus, rows > 0 ? rows : 1);
  const int64_t most = ceil_div(vectors, kThreads);
  if (want > most) want = most;
  if (k > 0 && want > kList / k) want = kList / k;
  if (rows * 4 > BSG_KV_COUNTER_BYTES) want = 1;
  Shape s;
  s.split_vectors = ceil_div(vectors, want);
  s.splits = (int32_t)ceil_div(vectors, s.split_vectors);
  return s;
}

int per_vector(int dtype) { return dtype == BSG_F32 ? 4 : 8; }

int64_t workspace_bytes(const Shape& s, int64_t rows, int32_t k) {
  return s.splits <= 1 ? 0 : BSG_KV_COUNTER_BYTES + rows * s.splits * (16 + 8 * (int64_t)k);
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
  return workspace_bytes(shape_of(rows, vocab, k, per_vector(dtype), cu_count), rows, k);
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
  const Shape s = shape_of(rows, vocab, k, per_vector(dtype), cu_count);
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
  // one launch takes 65535 rows
  for (int64_t r = 0; r < rows; r += 65535) {
    const int64_t n = rows - r < 65535 ? rows - r : 65535;
    p.x = (const uint8_t*)logits + r * row_stride * (int64_t)es;
    p.tokens = tokens + r;
    p.logprob = logprob + r;
    p.entropy = entropy + r;
    p.top_ids = k > 0 ? top_ids + r * k : nullptr;
    p.top_logprobs = k > 0 ? top_logprobs + r * k : nullptr;
    const dim3 grid((unsigned)s.splits, (unsigned)n);
    if (dtype == BSG_F16)
      hipLaunchKernelGGL(bsg_token_logprobs_kernel<_Float16>, grid, dim3(kThreads), 0, st, p);
    else if (dtype == BSG_BF16)
      hipLaunchKernelGGL(bsg_token_logprobs_kernel<__bf16>, grid, dim3(kThreads), 0, st, p);
    else
      hipLaunchKernelGGL(bsg_token_logprobs_kernel<float>, grid, dim3(kThreads), 0, st, p);
  }
  return launch_status("bsg_token_logprobs");
}
