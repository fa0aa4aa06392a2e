// kv_quant.hpp — how numbers come into the 8-bit cache: a page's scale, rounding to e4m3, and the transposes
// between tokens of channels (as they come) and channels of tokens (as the values lie).
#pragma once

#include "serve.hpp"

namespace bsgk {

// Bytes b of the four dwords a quad's lanes hold, to lane b of the quad: the 4 x 4 byte transpose.
__device__ __forceinline__ uint32_t quad_transpose(uint32_t w, int i) {
  const uint32_t w0 = __builtin_amdgcn_mov_dpp(w, 0x00, 0xf, 0xf, true);
  const uint32_t w1 = __builtin_amdgcn_mov_dpp(w, 0x55, 0xf, 0xf, true);
  const uint32_t w2 = __builtin_amdgcn_mov_dpp(w, 0xaa, 0xf, 0xf, true);
  const uint32_t w3 = __builtin_amdgcn_mov_dpp(w, 0xff, 0xf, 0xf, true);
  const uint32_t sel = (uint32_t)i * 0x0101u + 0x0400u;  // byte i of each of two words
  const uint32_t lo = __builtin_amdgcn_perm(w1, w0, sel) & 0xffffu;
  const uint32_t hi = __builtin_amdgcn_perm(w3, w2, sel) & 0xffffu;
  return lo | (hi << 16);
}

// The 4 x 4 transpose of four dwords over the four rows of 16 lanes.
__device__ __forceinline__ void row_transpose(uint32_t w[4]) {
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const auto r = __builtin_amdgcn_permlane32_swap(w[n], w[n + 2], false, false);
    w[n] = r[0], w[n + 2] = r[1];
  }
#pragma unroll
  for (int n = 0; n < 4; n += 2) {
    const auto r = __builtin_amdgcn_permlane16_swap(w[n], w[n + 1], false, false);
    w[n] = r[0], w[n + 1] = r[1];
  }
}

// x / scale to e4m3, rounded to nearest even: the product with a power of two is exact, infinities
// become the largest value, NaN stays.
__device__ __forceinline__ float in_range(float x) { return x != x ? x : fminf(fmaxf(x, -448.f), 448.f); }

__device__ __forceinline__ uint32_t to_e4m3(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(in_range(a), in_range(b), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(in_range(c), in_range(d), r, true);
}

// Four cached numbers under a new, larger scale.
__device__ __forceinline__ uint32_t rescale(uint32_t w, float ratio) {
  return to_e4m3(__builtin_amdgcn_cvt_f32_fp8((int)w, 0) * ratio, __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * ratio,
                 __builtin_amdgcn_cvt_f32_fp8((int)w, 2) * ratio, __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * ratio);
}

// The least power of two s in [2^-40, 2^80] with a <= 448 s, from the bits of a = 1.m x 2^e:
// 448 = 1.75 x 2^8.
__device__ __forceinline__ float scale_for(float a) {
  const int e = (int)((__builtin_bit_cast(uint32_t, a) + 0x1fffffu) >> 23) - 127 - 8;
  const int c = e < BSG_KV_SCALE_MIN_EXP ? BSG_KV_SCALE_MIN_EXP : e > BSG_KV_SCALE_MAX_EXP ? BSG_KV_SCALE_MAX_EXP : e;
  return __builtin_bit_cast(float, (uint32_t)(c + 127) << 23);
}

// The largest finite magnitude in the wave.  Magnitudes of either 16-bit type order as their bits do; only where
// infinities or NaN are among them are those taken out.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
template <typename T>
inline constexpr uint32_t kInfBits = 0x7c00u;
template <>
inline constexpr uint32_t kInfBits<__bf16> = 0x7f80u;

template <int X>
__device__ __forceinline__ u16x2 wave_max(u16x2 m) {
  m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, lane_xor<X>(__builtin_bit_cast(uint32_t, m))));
  if constexpr (X > 1) m = wave_max<X / 2>(m);
  return m;
}
template <typename T, int C>
__device__ __forceinline__ float largest_magnitude(const uint32_t x[C][8]) {
  u16x2 m = {0, 0};
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, x[c][i] & 0x7fff7fffu));
  m = wave_max<32>(m);
  uint32_t top = m.x > m.y ? m.x : m.y;
  if (top >= kInfBits<T>) {
    m = u16x2{0, 0};
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t w = x[c][i] & 0x7fff7fffu;
        const uint32_t lo = w & 0xffffu, hi = w >> 16;
        m = __builtin_elementwise_max(m, u16x2{(unsigned short)(lo < kInfBits<T> ? lo : 0u), (unsigned short)(hi < kInfBits<T> ? hi : 0u)});
      }
    m = wave_max<32>(m);
    top = m.x > m.y ? m.x : m.y;
  }
  return low_half<T>(top);
}

}  // namespace bsgk
