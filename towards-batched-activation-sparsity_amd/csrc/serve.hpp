// serve.hpp — what the serving operators' units share: the C ABI's error message, argument helpers,
// and small device primitives (16-bit element types, cross-lane sums, the hand-off of partials).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "bsgserve.h"

namespace bsgk {

// Sets the calling thread's bsg_last_error() message and returns `code` (bsgemm.hip).
int fail(int code, const char* fmt, ...);

inline int launch_status(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? BSG_OK : fail(BSG_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

// One launch takes fewer than 2^32 threads in x; past that it is cut short without an error.
constexpr int64_t kLaunchGroups = (1 << 24) - 1;  // of 256 threads

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline bool is_aligned(const void* p, unsigned n) { return ((uintptr_t)p & (n - 1)) == 0; }

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// By value: a bit cast of a vector's element in place reads its first one.
__device__ __forceinline__ float as_float(uint32_t w) { return __builtin_bit_cast(float, w); }

// Both halves of a 32-bit word of two 16-bit numbers, as fp32 (exact).
template <typename T>
__device__ __forceinline__ float low_half(uint32_t w);
template <typename T>
__device__ __forceinline__ float high_half(uint32_t w);
template <>
__device__ __forceinline__ float low_half<_Float16>(uint32_t w) {
  return (float)__builtin_bit_cast(f16x2, w).x;
}
template <>
__device__ __forceinline__ float high_half<_Float16>(uint32_t w) {
  return (float)__builtin_bit_cast(f16x2, w).y;
}
template <>
__device__ __forceinline__ float low_half<__bf16>(uint32_t w) {
  return __builtin_bit_cast(float, w << 16);
}
template <>
__device__ __forceinline__ float high_half<__bf16>(uint32_t w) {
  return __builtin_bit_cast(float, w & 0xffff0000u);
}

// The value of lane ^ X.
template <int X>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
  if constexpr (X == 1) return __builtin_amdgcn_mov_dpp(v, 0xb1, 0xf, 0xf, true);   // quad_perm 1 0 3 2
  if constexpr (X == 2) return __builtin_amdgcn_mov_dpp(v, 0x4e, 0xf, 0xf, true);   // quad_perm 2 3 0 1
  if constexpr (X == 4) {                                                           // 7 - i, then 3 - i in quads
    v = __builtin_amdgcn_mov_dpp(v, 0x141, 0xf, 0xf, true);
    return __builtin_amdgcn_mov_dpp(v, 0x1b, 0xf, 0xf, true);
  }
  if constexpr (X == 8) return __builtin_amdgcn_mov_dpp(v, 0x128, 0xf, 0xf, true);  // row_ror:8
  if constexpr (X == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return threadIdx.x & 16 ? r[0] : r[1];
  }
  if constexpr (X == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return threadIdx.x & 32 ? r[0] : r[1];
  }
}
template <int X>
__device__ __forceinline__ float lane_xor(float v) {
  return as_float(lane_xor<X>(__builtin_bit_cast(uint32_t, v)));
}
template <int X>
__device__ __forceinline__ uint64_t lane_xor(uint64_t v) {
  return (uint64_t)lane_xor<X>((uint32_t)(v >> 32)) << 32 | lane_xor<X>((uint32_t)v);
}

// Partials cross work-groups with agent-scope relaxed atomics (device-coherent, with no fence that
// would write back and invalidate a whole L2): every wave waits for its stores, the work-group
// meets in a barrier, and one thread counts the arrival.
__device__ __forceinline__ void hand_store(uint64_t* p, uint64_t v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t hand_load(const uint64_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// The same 16 bytes at a time: a buffer's loads and stores with the scope bit of an agent (sc1).
constexpr int kAgent = 16;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t hand_buffer(const void* base, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00020000);
}
__device__ __forceinline__ void hand_store16(__amdgpu_buffer_rsrc_t r, int off, f32x4 v) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), r, off, 0, kAgent);
}
__device__ __forceinline__ f32x4 hand_load16(__amdgpu_buffer_rsrc_t r, int off) {
  return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, kAgent));
}
__device__ __forceinline__ f32x2 hand_load8(__amdgpu_buffer_rsrc_t r, int off) {
  return __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, kAgent));
}
__device__ __forceinline__ void hand_publish() {
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
}
__device__ __forceinline__ uint32_t hand_arrive(uint32_t* c) {
  return __hip_atomic_fetch_add(c, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void hand_reset(uint32_t* c) {
  __hip_atomic_store(c, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

}  // namespace bsgk
