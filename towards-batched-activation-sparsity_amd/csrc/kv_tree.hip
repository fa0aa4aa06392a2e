// kv_tree.hip — attention of a tree of drafted tokens over the 8-bit paged cache (include/bsgdraft.h).
//
// A row sees all tokens before the tree, and of the tree its own node and its ancestors, which each wave works out
// once, one bit for each of 64 nodes.  Only the last steps hold nodes, so only they look at the bits.  Up to 32 rows of a
// cached head go to kv_attention.hpp's kernel, more to the one below; the arithmetic is the same.  HBM bounds the first: 64
// trees of up to 16 nodes, contexts to 1500 tokens, 32 heads (509 MB), 95 us, 5.3 TB/s (three waves a SIMD instead of two: 113).

#include "bsgdraft.h"
#include "kv_attention.hpp"

namespace {

// How the second kernel's work is cut.  A unit is a tile of rows of one cached head of one sequence, a step 64 of the
// tokens that it sees.  Trees of a batch have few units of unequal lengths, so the steps of all units, one after
// the other, are dealt out evenly to at most `groups` work-groups, whoever's they are: a work-group finishes the unit that
// the one before began, does some whole ones and begins another.  What it has of a unit that is not all its own it leaves as
// a part; a second launch joins the parts.
struct TreeParams {
  AttnParams a;
  int32_t tiles, groups, rows;  // of a cached head, at most; work-groups (0: one for each unit, and no parts); sequences
  int32_t sorted;               // without a deal: long sequences first
  uint2* units;   // [sequence][head][tile]: the first work-group that has a part, how many have
  float* parts;   // [work-group][2]: of the unit that it finishes, of the one that it begins
};
constexpr int kStep = 64;       // tokens
constexpr int kLeastSteps = 4;  // of a work-group
constexpr int kMostRows = 256;  // sequences that are dealt out: as many as a work-group has threads
constexpr int kRows = 128, kSmallRows = 64;  // of a tile, and of a small one
// What weighs as much where steps are dealt out: a step of a tile (2.6 us beside another work-group), one of a small tile (1.6),
// and what a unit costs a work-group beside its steps.  With nothing for the last, us: one sequence of 40 rows and 800
// tokens 23, 18.7 with it; 8 x 8 heads x 100 rows of up to 3000 tokens 36, 32; 16 x 8 x 240 rows of up to 6001 94, 91.
constexpr uint32_t kWeight = 8, kSmallWeight = 5, kBegin = 24;
// When they are dealt out: fewer units than kDealUnits a compute unit, of more than kDealTokens tokens.  A work-group for
// each unit / dealt out, us: 256 units of up to 2000 tokens 43 / 39, 512 of them 53 / 62, 1024 98 / 100; 8 sequences x 8 heads
// x 100 rows of up to 3000 tokens 83 / 32, 16 x 8 x 240 rows of up to 6001 160 / 90; 32 units of up to 800 tokens 23 / 19, of
// 600 21 / 19, 128 of them 22 / 25, of 300 17 / 22.
constexpr int kDealUnits = 2;
constexpr int kDealTokens = 768;
// Work-groups for each unit begin with the longest sequences where not all have room at once (two a compute unit have) and there
// are fewer than kSortUnits a compute unit, so that the last ones to begin matter.  As they come / sorted, us: 1024 units of up to
// 2000 tokens 99 / 82; 2048 of up to 1000 113 / 115; 512, which begin at once, 51 / 54 and 80 / 78.
constexpr int kSortUnits = 6;
// Two waves share a SIMD, and the older one goes first, so that it ends early and the other one has nobody beside it for the
// rest (at 60 and 100 us in the case below).  Every 2^kTurn cycles the other one has priority: 97 us in all, 102 without.
constexpr int kTurn = 14;

// A part: [16 rows][16 channels][lane] accumulators in the order the matrix unit leaves them, then base and sum of
// each row.
template <int D>
constexpr int part_floats(int rows) { return rows * (D + 2); }

// A sequence of the batch.
struct Branch {
  int64_t from;
  int slot, count, len, first;
};
__device__ __forceinline__ Branch branch_of(const AttnParams& p, int row) {
  Branch b;
  b.slot = p.slots ? p.slots[row] : row;
  int64_t to = (int64_t)(row + 1) * p.max_new;
  b.from = (int64_t)row * p.max_new;
  if (p.cu) b.from = p.cu[row], to = p.cu[row + 1];
  const bool fine = b.from >= 0 && b.from < to && to <= p.tokens;
  b.count = !fine ? 0 : (int)(to - b.from < p.max_new ? to - b.from : p.max_new);
  int len = b.slot >= 0 && b.slot < p.num_slots ? p.lengths[b.slot] : 0;
  const int most = p.max_pages << p.page_shift;
  b.len = len < 0 ? 0 : len > most ? most : len;
  b.first = fine ? b.len - (int)(to - b.from) : 0;
  return b;
}
// Steps of a unit, and units of a cached head.
__device__ __forceinline__ int steps_of(const Branch& b) {
  const int end = b.first + b.count;
  return b.count == 0 ? 0 : end <= kStep ? 1 : (end + kStep - 1) / kStep;
}
// The tiles of a cached head's rows, of ROWS each; where those are kRows and what is left is at most kSmallRows, the last one
// is a small one.
template <int ROWS>
__device__ __forceinline__ int tiles_of(const AttnParams& p, const Branch& b) { return (b.count * p.group + ROWS - 1) / ROWS; }
template <int ROWS>
__device__ __forceinline__ bool ends_small(const AttnParams& p, const Branch& b) {
  return ROWS == kSmallRows || ((b.count * p.group - 1) & (ROWS - 1)) < kSmallRows;
}
template <int ROWS>
constexpr uint32_t kTileWeight = ROWS == kSmallRows ? kSmallWeight : kWeight;
template <int ROWS>
__device__ __forceinline__ uint32_t weight_of(const AttnParams& p, const Branch& b) {  // of a step of all tiles of a head
  return b.count == 0 ? 0 : tiles_of<ROWS>(p, b) * kTileWeight<ROWS> - (ends_small<ROWS>(p, b) ? kTileWeight<ROWS> - kSmallWeight : 0);
}

// The sequence of work-group z where those of long sequences come first, of each 64.
__device__ __forceinline__ int longest_first(const AttnParams& p, int rows) {
  const int lane = threadIdx.x & 63, of = blockIdx.z & ~63, row = of + lane;
  int len = -1;
  if (row < rows) {
    const int slot = p.slots ? p.slots[row] : row;
    len = slot >= 0 && slot < p.num_slots ? p.lengths[slot] : 0;
    if (len < 0) len = 0;
  }
  int before = 0;
#pragma unroll 8
  for (int i = 0; i < 64; ++i) {
    const int other = __builtin_amdgcn_readlane(len, i);
    before += other > len || (other == len && i < lane);
  }
  return of + __builtin_ctzll(__ballot(before == (int)(blockIdx.z & 63)));
}

// A work-group of four waves has a tile of rows, each wave 32 of them, and takes the tokens they see 64 at a time,
// brought once straight into LDS in the bytes they have in memory, a pair of steps ahead (the waves meet once a pair, not once
// a step: 1024 units of up to 2000 tokens 98 us, 101).  In a small tile the other two waves have the same rows and the second
// half of each step's tokens; the halves meet in LDS at the end.
// What two waves a SIMD hide of the softmax between the products bounds it: of a step of a wave (3300 cycles of its SIMD) the
// vector unit is at work for some 2000 and the matrix unit for 1000.  16 sequences of up to 6001 tokens, 8 heads x up to 240 rows,
// 43 GFLOP: 91 us, of which 10 are the join's, 8 come before a work-group's first step and 7 are memory's.
template <typename T, int D, int ROWS>
__global__ __launch_bounds__(256, 2) void bsg_kv_tree_kernel(TreeParams tp) {
  const AttnParams& p = tp.a;
  constexpr int C = D / 64, DT = D / 16, RT = 2;
  typedef typename Elem<T>::x8 x8;
  constexpr int TILE = 2 * C * 64;  // 16-byte pieces of a 16-token tile, keys then values
  // what the work-groups agree on about the sequences: their weights, those before them, and what they are
  __shared__ uint32_t s_scan[4], s_weight[kMostRows], s_before[kMostRows];
  __shared__ Branch s_branch[kMostRows];
  __shared__ int32_t s_row;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, g = lane >> 4;

  const uint32_t slot = __builtin_amdgcn_s_getreg(4 | 0 << 6 | 3 << 11);  // the wave's place on its SIMD

  uint32_t group = 0, per = 1, pos = 0, stop = 1;  // the weights that are the work-group's
  if (tp.groups > 0) {
    uint32_t mine = 0, total = 0;
    if ((int)threadIdx.x < tp.rows) {
      const Branch b = branch_of(p, threadIdx.x);
      s_branch[threadIdx.x] = b;
      mine = (steps_of(b) * weight_of<ROWS>(p, b) + tiles_of<ROWS>(p, b) * kBegin) * p.kv_heads;
    }
    uint32_t upto = mine;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const uint32_t o = __shfl_up(upto, m);
      if (lane >= m) upto += o;
    }
    if (lane == 63) s_scan[wave] = upto;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < wave) upto += s_scan[w];
      total += s_scan[w];
    }
    total = __builtin_amdgcn_readfirstlane(total);
    s_weight[threadIdx.x] = mine, s_before[threadIdx.x] = upto - mine;
    per = (total + tp.groups - 1) / tp.groups;
    if (per < kLeastSteps * kTileWeight<ROWS>) per = kLeastSteps * kTileWeight<ROWS>;
    // Those that follow each other, which often read the same keys and values for other rows, run on one die and share its
    // L2 (8 x 8 heads x 100 rows of up to 3000 tokens: 35 us, in the launch's order 36; 240 rows of up to 6001 101, 102).
    const uint32_t on_die = ((total + per - 1) / per + 7) / 8;
    if (blockIdx.x / 8 >= on_die) return;
    group = blockIdx.x % 8 * on_die + blockIdx.x / 8;
    const uint64_t begin = (uint64_t)group * per;
    if (begin >= total) return;
    pos = (uint32_t)begin;
    stop = total - pos > per ? pos + per : total;
  }
  const int own_row = __builtin_amdgcn_readfirstlane(tp.sorted ? longest_first(p, tp.rows) : (int)blockIdx.z);
  while (pos < stop) {
    int row, head, rt, step0 = 0, step1, steps;
    uint32_t unit_at = 0, weight = 1;  // where the unit's weights begin, the weight of its steps
    Branch b;
    if (tp.groups > 0) {
      __syncthreads();
      if (pos - s_before[threadIdx.x] < s_weight[threadIdx.x]) s_row = threadIdx.x;
      __syncthreads();
      row = __builtin_amdgcn_readfirstlane(s_row);
      const uint32_t in_row = pos - __builtin_amdgcn_readfirstlane(s_before[row]);
      b.from = __builtin_amdgcn_readfirstlane((int)s_branch[row].from);  // tokens are below 2^31
      b.slot = __builtin_amdgcn_readfirstlane(s_branch[row].slot), b.count = __builtin_amdgcn_readfirstlane(s_branch[row].count);
      b.len = __builtin_amdgcn_readfirstlane(s_branch[row].len), b.first = __builtin_amdgcn_readfirstlane(s_branch[row].first);
      steps = steps_of(b);
      const uint32_t of_head = steps * weight_of<ROWS>(p, b) + tiles_of<ROWS>(p, b) * kBegin, of_tile = steps * kTileWeight<ROWS> + kBegin;
      head = in_row / of_head;
      const uint32_t in_head = in_row - head * of_head;
      rt = in_head / of_tile;
      weight = rt == tiles_of<ROWS>(p, b) - 1 && ends_small<ROWS>(p, b) ? kSmallWeight : kTileWeight<ROWS>;
      unit_at = pos - (in_head - rt * of_tile) + kBegin;
      // step j is the work-group's that has the weight unit_at + j weight
      step0 = pos <= unit_at ? 0 : (pos - unit_at + weight - 1) / weight;
      step1 = stop <= unit_at ? 0 : (stop - unit_at + weight - 1) / weight;
      if (step1 > steps) step1 = steps;
      pos = step1 == steps ? unit_at + steps * weight : stop;
      if (step0 >= step1) continue;
    } else {
      row = own_row, head = blockIdx.x / tp.tiles;
      b = branch_of(p, row);
      rt = blockIdx.x - head * tp.tiles;
      step1 = steps = steps_of(b);
      if (rt >= tiles_of<ROWS>(p, b)) return;
      pos = stop;
    }
    const bool whole = step1 - step0 == steps;
    if (tp.groups > 0 && step0 == 0 && threadIdx.x == 0)
      tp.units[((int64_t)row * p.kv_heads + head) * tp.tiles + rt] =
          make_uint2(group, whole ? 0u : (unit_at + (uint32_t)(steps - 1) * weight) / per - group + 1);
    const int64_t from = b.from;
    const int first = b.first;
    const int rows = b.count * p.group - rt * ROWS, used = rows < ROWS ? rows : ROWS;
    const auto sees_until = [&](int r) {  // past the last token that row r of the tile sees
      const int n = first + (rt * ROWS + r) / p.group + 1;
      return n < 0 ? 0 : n;
    };
    const int end = sees_until(used - 1);
    const int t_begin = step0 * kStep;
    const int t_end = step1 * kStep < end ? step1 * kStep : end;
    const int parent = load_parent(p.parents, from, b.count, lane);
    const float scale2 = __builtin_fabsf(p.scale2);

    const int32_t* const table = p.table + (int64_t)(b.slot < 0 || b.slot >= p.num_slots ? 0 : b.slot) * p.table_stride;
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
      const int64_t at_bytes = n < 16 ? tiles.at : next_at;
      const int at = 4 * n + wave & 63;
      const int lo = __builtin_amdgcn_readlane((int)at_bytes, at), hi = __builtin_amdgcn_readlane((int)(at_bytes >> 32), at);
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

    // the cache's chain of loads (pages, scales, tiles) before what is only wanted at the first step
    if (t_begin < t_end) {
      load_pages(t_begin);
      load_scales(t_begin);
      tiles.at = next_at;
      issue(std::integral_constant<int, 0>{}, 0);
      issue(std::integral_constant<int, 1>{}, 1);
      turn_pages();
    }
    const uint64_t lineage = lineage_of(parent, lane);
    const auto run = [&](auto row_groups) {  // of 32 rows
      constexpr int RG = decltype(row_groups)::value, TG = 4 / RG, NT = 4 / TG;  // NT: a wave's 16-token tiles of a step
      const int rg = wave % RG, tg = wave / RG;
      // this wave's rows: 32 rg .. +31
      const int w_used = used - 32 * rg < 32 ? used - 32 * rg : 32;
      const int w_end = w_used > 0 ? sees_until(32 * rg + w_used - 1) : 0;  // past what its last row sees
      const int w_all = w_used > 0 && first > 0 ? first : 0;                // what all of them see

      x8 qf[RT][2 * C];
      Sight<true> sees[RT];
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const int r = 32 * rg + 16 * i + col;
        const int rr = rt * ROWS + r, tok = rr / p.group, h = rr - tok * p.group;
        const bool on = r < used;
        const uint64_t mask = from_lane(lineage, tok & 63);
        sees[i] = on ? Sight<true>{first, mask} : Sight<true>::none();
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

      f32x4 acc[RT][DT];
      float base[RT], l[RT];  // -inf: no token seen
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        base[i] = -__builtin_inff(), l[i] = 0.f;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[i][d] = f32x4{0.f, 0.f, 0.f, 0.f};
      }

      bool started = false;  // every row has a base, and one that is near 0
      const auto take = [&](auto stage, int step_at) {
        const u32x4* const kv = prefill_stage<D, decltype(stage)::value>() + lane + tg * NT * TILE;
        const int first_tile = ((step_at - t_begin) / 16 & 63) + tg * NT;
        const int t0 = step_at + 16 * NT * tg;  // the first of the wave's tokens
        f32x4 s[RT][NT];
        float ks[NT], lv[NT], iv[NT];
        bool there[NT], all_there = true;
#pragma unroll
        for (int a = 0; a < NT; ++a) {
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
        const bool partial = t0 + 16 * NT > w_all || !all_there;
        if (partial) {
#pragma unroll
          for (int a = 0; a < NT; ++a)
#pragma unroll
            for (int i = 0; i < RT; ++i) {
              const uint32_t four = there[a] ? sees[i].four(t0 + 16 * a + 4 * g) : 0u;
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if ((four >> j & 1u) == 0) s[i][a][j] = -__builtin_inff();
            }
        }
        // Weights against the base so far; only where four of them together outgrow fp16 (or a row has no
        // base yet, or none near 0) is a new one looked for.  Against a new base, and one that is not near 0, the score is rounded
        // first, so that the maximum's weight is 2^13 or 1 however far it is, and equal scores weigh the same; otherwise both
        // come in one step.
        f16x8 pf[RT][NT / 2];
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          float e[NT][4], sum[NT], top = 0.f;
          const auto weigh = [&](auto exactly) {
            const float off_base = base[i] == -__builtin_inff() ? 0.f : base[i];
            top = 0.f;
#pragma unroll
            for (int a = 0; a < NT; ++a) {
              const float off = lv[a] - off_base;
#pragma unroll
              for (int j = 0; j < 4; ++j)
                e[a][j] = __builtin_amdgcn_exp2f(decltype(exactly)::value ? __builtin_fmaf(s[i][a][j], ks[a], lv[a]) - off_base
                                                                          : __builtin_fmaf(s[i][a][j], ks[a], off));
              sum[a] = (e[a][0] + e[a][1]) + (e[a][2] + e[a][3]);
              top = fmaxf(top, sum[a]);
            }
          };
          weigh(std::false_type{});
          if (!started || __any(top > kMostWeight)) {
            float mx = -__builtin_inff();
#pragma unroll
            for (int a = 0; a < NT; ++a) {
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
          uint32_t w[2 * NT];
#pragma unroll
          for (int a = 0; a < NT; ++a) {
            l[i] = __builtin_fmaf(sum[a], iv[a], l[i]);
            w[2 * a] = Elem<_Float16>::pack(e[a][0], e[a][1]), w[2 * a + 1] = Elem<_Float16>::pack(e[a][2], e[a][3]);
          }
#pragma unroll
          for (int n = 0; n < NT / 2; ++n)
            pf[i][n] = __builtin_bit_cast(f16x8, u32x4{w[4 * n], w[4 * n + 1], w[4 * n + 2], w[4 * n + 3]});
        }
        if (!started)
          started = !partial && !__any(!(__builtin_fabsf(base[0]) < kNearScore) || !(__builtin_fabsf(base[1]) < kNearScore));
#pragma unroll
        for (int n = 0; n < NT / 2; ++n) {
#pragma unroll
          for (int c = 0; c < C; ++c) {
            u32x4 v[2] = {kv[2 * n * TILE + (C + c) * 64], kv[(2 * n + 1) * TILE + (C + c) * 64]};
            if (partial) {
              uint32_t nan = 0;
#pragma unroll
              for (int a = 0; a < 2; ++a) {
                v[a] &= there[2 * n + a] ? byte_mask(t_end - (t0 + 32 * n + 16 * a + 4 * g)) : 0u;
                nan |= nan_bytes(v[a].x) | nan_bytes(v[a].y) | nan_bytes(v[a].z) | nan_bytes(v[a].w);
              }
              if (__any(nan != 0)) nan_values<RT, true>(v, t0 + 32 * n + 4 * g, sees, &acc[0][4 * c], DT);
            }
#pragma unroll
            for (int d = 0; d < 4; ++d) {
              const f16x8 x = widen<_Float16>(v[0][d], v[1][d]);
#pragma unroll
              for (int i = 0; i < RT; ++i) acc[i][4 * c + d] = Elem<_Float16>::mfma(x, pf[i][n], acc[i][4 * c + d]);
            }
          }
        }
      };

      if (t_begin < t_end) {
        int n = 0;
        for (int t0 = t_begin; t0 < t_end; t0 += 4 * kStep)
          [&]<int... I>(std::integer_sequence<int, I...>) {
            (..., [&](auto half) {
              constexpr int S = 2 * decltype(half)::value;
              const int t = t0 + S * kStep;
              // this pair's pieces have arrived for every wave, and every wave has read the pair's before
              vmem_wait<0>();
              __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
              asm volatile("" ::: "memory");
              __builtin_amdgcn_s_barrier();
              asm volatile("" ::: "memory");
              __builtin_amdgcn_sched_barrier(0);
              if (n == 8) load_pages(t + 8 * kStep);
              if (n == 10) load_scales(t + 6 * kStep);
              issue(std::integral_constant<int, (S + 2) % 4>{}, n + 2);
              issue(std::integral_constant<int, (S + 3) % 4>{}, n + 3);
              __builtin_amdgcn_sched_barrier(0);
              if (((uint32_t)(__builtin_readcyclecounter() >> kTurn) ^ slot) & 1) __builtin_amdgcn_s_setprio(1);
              else __builtin_amdgcn_s_setprio(0);
              if (t < w_end && t < t_end) take(std::integral_constant<int, S>{}, t);
              if (t + kStep < w_end && t + kStep < t_end) take(std::integral_constant<int, S + 1>{}, t + kStep);
              if ((n += 2) == 16) n = 0, turn_pages();
            }(std::integral_constant<int, I>{}));
          }(std::make_integer_sequence<int, 2>{});
        vmem_wait<0>();  // nothing is on its way into LDS any more
      }
#pragma unroll
      for (int i = 0; i < RT; ++i) l[i] = column_sum(l[i]);

      if constexpr (TG == 2) {  // the second halves come over, 16 rows of a wave at a time
        f32x4* const s_half = (f32x4*)prefill_stage<D, 0>();  // [rg][channels / 16][lane]
        f32x2* const s_ml = (f32x2*)prefill_stage<D, 1>();    // [rg][lane]
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          __syncthreads();
          if (tg == 1) {
#pragma unroll
            for (int d = 0; d < DT; ++d) s_half[(rg * DT + d) * 64 + lane] = acc[i][d];
            s_ml[rg * 64 + lane] = f32x2{base[i], l[i]};
          }
          __syncthreads();
          if (tg == 0) {
            const f32x2 ml = s_ml[rg * 64 + lane];
            const float top = fmaxf(base[i], ml.x);
            const float mine = base[i] == top ? 1.f : __builtin_amdgcn_exp2f(base[i] - top);
            const float theirs = ml.x == top ? 1.f : __builtin_amdgcn_exp2f(ml.x - top);
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[i][d] = acc[i][d] * mine + s_half[(rg * DT + d) * 64 + lane] * theirs;
            l[i] = l[i] * mine + ml.y * theirs, base[i] = top;
          }
        }
      }
      if (tg == 0) {
        if (whole) {
#pragma unroll
          for (int i = 0; i < RT; ++i) {
            const int r = 32 * rg + 16 * i + col, rr = rt * ROWS + r, tok = rr / p.group, h = head * p.group + rr - tok * p.group;
            if (r < used) {
              const bool nothing = l[i] == 0.f;
              const float inv = nothing ? 0.f : 1.f / l[i];
              uint16_t* const at = p.out + (from + tok) * p.o_st + (int64_t)h * p.o_sh + 4 * g;
#pragma unroll
              for (int d = 0; d < DT; ++d)
                *(u32x2*)(at + 16 * d) = u32x2{Elem<T>::pack(acc[i][d][0] * inv, acc[i][d][1] * inv),
                                               Elem<T>::pack(acc[i][d][2] * inv, acc[i][d][3] * inv)};
              if (p.lse && g == 0)
                p.lse[(from + tok) * ((int64_t)p.kv_heads * p.group) + h] =
                    nothing ? -__builtin_inff() : (base[i] + __builtin_amdgcn_logf(l[i])) * (1.f / kLog2e);
            }
          }
        } else {
          float* const part = tp.parts + (int64_t)(2 * group + (step0 == 0)) * part_floats<D>(ROWS);
          int l0 = lane;  // whose offsets are not worth registers all along
          asm volatile("" : "+v"(l0));
#pragma unroll
          for (int i = 0; i < RT; ++i) {
#pragma unroll
            for (int d = 0; d < DT; ++d) *(f32x4*)(part + (((2 * rg + i) * DT + d) * 64 + l0) * 4) = acc[i][d];
            if (l0 < 16) *(f32x2*)(part + ROWS * D + 2 * (32 * rg + 16 * i + l0)) = f32x2{base[i], l[i]};
          }
        }
      }
    };
    if constexpr (ROWS == kSmallRows) run(std::integral_constant<int, 2>{});
    else if (used <= kSmallRows) run(std::integral_constant<int, 2>{});
    else run(std::integral_constant<int, 4>{});
  }
}

// The parts of the units that several work-groups had, joined in order: a wave has 16 channels of 16 rows (all channels of them:
// 81 us where the two launches now take 67, one tree of 60 nodes and 30000 tokens).
template <typename T, int D, int ROWS>
__global__ __launch_bounds__(256) void bsg_kv_tree_join_kernel(TreeParams tp) {
  const AttnParams& p = tp.a;
  constexpr int DT = D / 16, BLOCKS = ROWS / 16, BATCH = 4;
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int64_t job = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t unit = job / (BLOCKS * DT);
  const int in_unit = (int)(job - unit * (BLOCKS * DT)), block = in_unit / DT, d = in_unit % DT;
  if (unit >= (int64_t)tp.rows * p.kv_heads * tp.tiles) return;
  const uint2 had = tp.units[unit];  // on its way beside the sequence; not looked at where that has no such rows
  const int row = (int)(unit / (p.kv_heads * tp.tiles)), in_row = (int)(unit - (int64_t)row * p.kv_heads * tp.tiles);
  const int head = in_row / tp.tiles, rt = in_row - head * tp.tiles;
  const Branch b = branch_of(p, row);
  if (b.count * p.group <= rt * ROWS + 16 * block || had.y == 0) return;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  float top = -__builtin_inff(), sum = 0.f;
  for (uint32_t s0 = 0; s0 < had.y; s0 += BATCH) {
    f32x2 ml[BATCH];
    f32x4 v[BATCH];
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      const uint32_t s = s0 + j < had.y ? s0 + j : had.y - 1;
      const float* const from = tp.parts + (int64_t)(2 * (had.x + s) + (s == 0)) * part_floats<D>(ROWS);
      ml[j] = *(const f32x2*)(from + ROWS * D + 2 * (16 * block + col));
      v[j] = *(const f32x4*)(from + ((block * DT + d) * 64 + lane) * 4);
    }
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      if (s0 + j >= had.y) continue;
      const float next = fmaxf(top, ml[j].x);
      const float mine = top == next ? 1.f : __builtin_amdgcn_exp2f(top - next);
      const float theirs = ml[j].x == next ? 1.f : __builtin_amdgcn_exp2f(ml[j].x - next);
      acc = acc * mine + v[j] * theirs;
      sum = sum * mine + ml[j].y * theirs, top = next;
    }
  }
  const int rr = rt * ROWS + 16 * block + col, tok = rr / p.group, h = head * p.group + rr - tok * p.group;
  if (tok >= b.count) return;
  const bool nothing = sum == 0.f;
  const float inv = nothing ? 0.f : 1.f / sum;
  uint16_t* const at = p.out + (b.from + tok) * p.o_st + (int64_t)h * p.o_sh + 16 * d + 4 * g;
  *(u32x2*)at = u32x2{Elem<T>::pack(acc[0] * inv, acc[1] * inv), Elem<T>::pack(acc[2] * inv, acc[3] * inv)};
  if (p.lse && g == 0 && d == 0)
    p.lse[(b.from + tok) * ((int64_t)p.kv_heads * p.group) + h] =
        nothing ? -__builtin_inff() : (top + __builtin_amdgcn_logf(sum)) * (1.f / kLog2e);
}

// A cached head's rows past which the second kernel runs.  First / second, us: 24 rows 22 / 25, 32 rows 67 / 75 and 41 / 42; 48
// rows of 16 sequences 75 / 50, 64 of 64 160 / 113; 40 rows of one sequence 18 / 19.
constexpr int kTileRows = 32;

// How a call is cut.  shape: of the first kernel; for the second one rows are the tile's and `groups` work-groups share
// the steps, or, 0, each unit has one.
struct Cut {
  Shape shape;
  int32_t groups, sorted;
  int64_t units, bytes;  // of the second kernel: units at most; of the workspace
};
Cut cut_of(int32_t rows, const bsg_kv_cache* cache, int32_t group, int32_t max_new, int64_t max_len, int32_t cus) {
  Cut c;
  Shape& s = c.shape;
  const int32_t kv_heads = cache->n_heads, d = cache->head_dim;
  const int64_t per_head = (int64_t)max_new * group;
  // past kSmallRows a tile is a small one only at the end; all small, us: 240 rows 111, not 90; 100 of 64 sequences 96, not 79, of 8
  // 30, not 32.  Below, the kernel without the large ones: 19, not 21 (one sequence of 40 rows), 27.5, not 29 (8 of 64).
  s.rows = per_head <= 16 ? 16 : per_head <= kTileRows ? 32 : per_head <= kSmallRows ? kSmallRows : kRows;
  s.row_tiles = (int32_t)ceil_div(per_head, s.rows);
  const int64_t tiles = (int64_t)rows * kv_heads * s.row_tiles;
  c.groups = 0, c.units = tiles;
  c.sorted = rows > 1 && tiles > (int64_t)kDealUnits * cus && tiles < (int64_t)kSortUnits * cus;
  if (max_len < 1) max_len = 1;
  s.chunk = (int32_t)(ceil_div(max_len, 128) * 128), s.splits = 1;
  if (s.rows >= kSmallRows) {
    // all weights, of rows as long as a table's can be, are counted in 32 bits
    const int64_t most = ceil_div((int64_t)cache->max_pages * cache->page_size, kStep);
    if (rows <= kMostRows && tiles < (int64_t)kDealUnits * cus && max_len > kDealTokens && tiles * (most * kWeight + kBegin) <= 0x7fffffff)
      c.groups = (int32_t)(ceil_div(2 * (int64_t)cus, 8) * 8);
    c.bytes = c.groups == 0 ? 0 : BSG_KV_COUNTER_BYTES + ceil_div(tiles * 8, 256) * 256 + (int64_t)c.groups * 2 * s.rows * (d + 2) * 4;
    return c;
  }
  int64_t want = ceil_div((int64_t)2 * cus, tiles > 0 ? tiles : 1);
  if (want > kMaxSplits) want = kMaxSplits;
  if (want > ceil_div(max_len, 256)) want = ceil_div(max_len, 256);
  if (tiles * 4 > BSG_KV_COUNTER_BYTES) want = 1;
  s.chunk = (int32_t)(ceil_div(ceil_div(max_len, want), 128) * 128);
  s.splits = (int32_t)ceil_div(max_len, s.chunk);
  c.bytes = workspace_bytes(s, rows, kv_heads, d);
  return c;
}

template <typename T, int D, int ROWS>
void launch_tiles(const TreeParams& t, const Cut& c, hipStream_t st) {
  if (c.groups == 0) {
    const dim3 grid((unsigned)(t.a.kv_heads * t.tiles), 1, (unsigned)t.rows);
    hipLaunchKernelGGL((bsg_kv_tree_kernel<T, D, ROWS>), grid, dim3(256), 0, st, t);
    return;
  }
  hipLaunchKernelGGL((bsg_kv_tree_kernel<T, D, ROWS>), dim3((unsigned)c.groups), dim3(256), 0, st, t);
  const int64_t waves = c.units * (ROWS / 16) * (D / 16);
  hipLaunchKernelGGL((bsg_kv_tree_join_kernel<T, D, ROWS>), dim3((unsigned)ceil_div(waves, 4)), dim3(256), 0, st, t);
}

template <typename T, int D>
void launch(const AttnParams& p, const Cut& c, int32_t rows, hipStream_t st) {
  const Shape& s = c.shape;
  if (s.rows <= 32) {
    const dim3 grid((unsigned)(p.kv_heads * s.row_tiles), (unsigned)s.splits, (unsigned)rows);
    if (s.rows == 16) hipLaunchKernelGGL((bsg_kv_attention_kernel<T, D, 1, true>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((bsg_kv_attention_kernel<T, D, 2, true>), grid, dim3(256), 0, st, p);
    return;
  }
  TreeParams t;
  t.a = p;
  t.tiles = s.row_tiles, t.groups = c.groups, t.rows = rows, t.sorted = c.sorted;
  t.units = (uint2*)((uint8_t*)p.counters + BSG_KV_COUNTER_BYTES);
  t.parts = (float*)((uint8_t*)t.units + ceil_div(c.units * 8, 256) * 256);
  if (s.rows == kSmallRows) launch_tiles<T, D, kSmallRows>(t, c, st);
  else launch_tiles<T, D, kRows>(t, c, st);
}

int check_nodes(int32_t max_new) {
  if (max_new > BSG_TREE_NODES) return fail(BSG_ERR_UNSUPPORTED, "%d nodes in a tree (at most %d)", max_new, BSG_TREE_NODES);
  return BSG_OK;
}

}  // namespace

extern "C" int64_t bsg_kv_tree_attention_workspace_bytes(const bsg_kv_cache* cache, int32_t rows, int32_t q_heads,
                                                         int32_t max_new, int64_t max_len, int32_t cu_count) {
  if (check_kv_cache(cache) || check_heads(cache, q_heads) || rows < 0 || max_new < 0 || check_nodes(max_new) || cu_count < 1)
    return -1;
  const int64_t most = (int64_t)cache->max_pages * cache->page_size;
  if (max_len <= 0 || max_len > most) max_len = most;
  return rows == 0 ? 0 : cut_of(rows, cache, q_heads / cache->n_heads, max_new, max_len, cu_count).bytes;
}

extern "C" int bsg_kv_tree_attention(const void* q, int64_t q_stride_t, int64_t q_stride_h, int64_t tokens,
                                     int32_t q_heads, const int32_t* parents, const bsg_kv_cache* cache,
                                     const int32_t* slots, int32_t rows, const int32_t* cu, int32_t max_new,
                                     int64_t max_len, float sm_scale, void* out, int64_t o_stride_t, int64_t o_stride_h,
                                     float* lse, int dtype, void* ws, int64_t ws_bytes, int32_t cu_count, void* stream) {
  const AttnCall c = {q, q_stride_t, q_stride_h, tokens, q_heads, cache, slots, rows, cu, max_new, sm_scale, out,
                      o_stride_t, o_stride_h, lse, dtype, ws, ws_bytes, cu_count};
  if (const int rc = check_call(c)) return rc;
  if (const int rc = check_nodes(max_new)) return rc;
  if (tokens == 0 || rows == 0 || max_new == 0) return BSG_OK;
  if (!parents) return fail(BSG_ERR_ARG, "parents is null");
  if (const int rc = check_tensors(c)) return rc;
  const int64_t most = (int64_t)cache->max_pages * cache->page_size;
  if (max_len <= 0 || max_len > most) max_len = most;
  const Cut cut = cut_of(rows, cache, q_heads / cache->n_heads, max_new, max_len, cu_count);
  AttnParams p;
  if (const int rc = call_params(c, cut.shape, cut.bytes, &p)) return rc;
  p.parents = parents;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == BSG_F16)
    cache->head_dim == 64 ? launch<_Float16, 64>(p, cut, rows, st) : launch<_Float16, 128>(p, cut, rows, st);
  else
    cache->head_dim == 64 ? launch<__bf16, 64>(p, cut, rows, st) : launch<__bf16, 128>(p, cut, rows, st);
  return launch_status("bsg_kv_tree_attention");
}
