// kv_attention.hip — attention of each sequence's newest tokens over its cached ones (include/bsgserve.h): the
// entry points, and how a call is cut.  The kernels are kv_attention.hpp's.

#include "kv_attention.hpp"

namespace {

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
  Sight<false> sees[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int r = 32 * wave + 16 * i + col;
    const int rr = rt * ROWS + r, tok = rr / p.group, h = rr - tok * p.group;
    const bool on = r < used;
    sees[i].until = on ? first + tok + 1 : 0;
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

  bool started = false;  // every row has a base, and one that is near 0
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
            if (t + j >= sees[i].until) s[i][a][j] = -__builtin_inff();
      }
    }
    // Weights against the base so far; only where four of them together outgrow fp16 (or a row has no
    // base yet, or none near 0) is a new one looked for.  The sums are wanted anyway: asking each weight took 590 us
    // instead of 566 for a prompt of 8192.  Against a new base, and one that is not near 0, the score is rounded first, so that
    // the maximum's weight is 2^13 or 1 however far it is, and equal scores weigh the same; otherwise both come in one step.
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
      started = !partial && !__any(!(__builtin_fabsf(base[0]) < kNearScore) || !(__builtin_fabsf(base[1]) < kNearScore));
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
          if (__any(nan != 0)) nan_values<RT, false>(v, t0 + 32 * b + 4 * g, sees, &acc[0][4 * c], DT);
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

template <typename T, int D>
void launch(const AttnParams& p, const Shape& s, dim3 grid, hipStream_t st) {
  switch (s.rows) {
    case 16: hipLaunchKernelGGL((bsg_kv_attention_kernel<T, D, 1, false>), grid, dim3(256), 0, st, p); break;
    case 32: hipLaunchKernelGGL((bsg_kv_attention_kernel<T, D, 2, false>), grid, dim3(256), 0, st, p); break;
    default: hipLaunchKernelGGL((bsg_kv_prefill_kernel<T, D>), grid, dim3(256), 0, st, p); break;
  }
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
  const AttnCall c = {q, q_stride_t, q_stride_h, tokens, q_heads, cache, slots, rows, cu, max_new, sm_scale, out,
                      o_stride_t, o_stride_h, lse, dtype, ws, ws_bytes, cu_count};
  if (const int rc = check_call(c)) return rc;
  if (tokens == 0 || rows == 0 || max_new == 0) return BSG_OK;
  if (const int rc = check_tensors(c)) return rc;
  const int64_t most = (int64_t)cache->max_pages * cache->page_size;
  if (max_len <= 0 || max_len > most) max_len = most;
  const Shape s = shape_of(rows, cache->n_heads, q_heads / cache->n_heads, max_new, max_len, cu_count);
  AttnParams p;
  if (const int rc = call_params(c, s, workspace_bytes(s, rows, cache->n_heads, cache->head_dim), &p)) return rc;
  const dim3 grid((unsigned)(cache->n_heads * s.row_tiles), (unsigned)s.splits, (unsigned)rows);
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == BSG_F16)
    cache->head_dim == 64 ? launch<_Float16, 64>(p, s, grid, st) : launch<_Float16, 128>(p, s, grid, st);
  else
    cache->head_dim == 64 ? launch<__bf16, 64>(p, s, grid, st) : launch<__bf16, 128>(p, s, grid, st);
  return launch_status("bsg_kv_attention");
}
