// Shared device code of the operators (tg_ops.hip): element types, unaligned vector access, cross-lane moves of a 64-lane wave.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tg {
namespace ops {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));

enum { kU8 = 0, kI8 = 1, kF32 = 2, kF16 = 3, kBF16 = 4 };

// 16 bytes at any address (gfx950 takes unaligned vector loads; a row of 13 or 200 bytes starts anywhere)
struct __attribute__((packed, aligned(1))) U128 { uint32_t w[4]; };
__device__ __forceinline__ v4i load16(const void* p) {
  const U128 u = *(const U128*)p;
  v4i r = {(int)u.w[0], (int)u.w[1], (int)u.w[2], (int)u.w[3]};
  return r;
}

struct bf16_t { uint16_t u; };
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(bf16_t v) { return __uint_as_float((uint32_t)v.u << 16); }

// one rounding, half to even; NaN stays NaN
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ _Float16 from_f32<_Float16>(float v) { return (_Float16)v; }
template <> __device__ __forceinline__ bf16_t from_f32<bf16_t>(float v) {
  const __bf16 b = (__bf16)v;
  bf16_t r;
  __builtin_memcpy(&r, &b, 2);
  return r;
}

// x as an unsigned key of the same order (x is not NaN; -0 counts as +0)
__device__ __forceinline__ uint32_t order_f32(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u ^ (uint32_t)(((int32_t)u >> 31) | (int32_t)0x80000000);
}
__device__ __forceinline__ float unorder_f32(uint32_t k) {
  return __uint_as_float(k ^ ((k & 0x80000000u) ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ uint64_t order_f64(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
  return u ^ (uint64_t)(((int64_t)u >> 63) | (int64_t)0x8000000000000000ull);
}
__device__ __forceinline__ double unorder_f64(uint64_t k) {
  return __longlong_as_double((long long)(k ^ ((k >> 63) ? 0x8000000000000000ull : ~0ull)));
}

// the value of lane (lane ^ M), on the vector unit (DPP inside a row of 16, permlane swaps across rows): no trip through LDS
template <int M> __device__ __forceinline__ uint32_t xor_lane(uint32_t v) {
  if constexpr (M == 1) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true);        // quad_perm 1,0,3,2
  else if constexpr (M == 2) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true);   // quad_perm 2,3,0,1
  else if constexpr (M == 4) {                                                                          // (i ^ 7) ^ 3
    const int t = __builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, true);                              // row_half_mirror
    return (uint32_t)__builtin_amdgcn_mov_dpp(t, 0x1B, 0xF, 0xF, true);                                 // quad_perm 3,2,1,0
  } else if constexpr (M == 8) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xF, 0xF, true);  // row_ror:8
  else if constexpr (M == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return (threadIdx.x & 16) ? r[0] : r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return (threadIdx.x & 32) ? r[0] : r[1];
  }
}
template <int M> __device__ __forceinline__ uint64_t xor_lane(uint64_t v) {
  return (uint64_t)xor_lane<M>((uint32_t)v) | ((uint64_t)xor_lane<M>((uint32_t)(v >> 32)) << 32);
}
template <int M> __device__ __forceinline__ float xor_lane(float v) { return __uint_as_float(xor_lane<M>(__float_as_uint(v))); }
template <int M> __device__ __forceinline__ double xor_lane(double v) {
  return __longlong_as_double((long long)xor_lane<M>((uint64_t)__double_as_longlong(v)));
}

// reductions over aligned groups of L lanes (L = 1, 2, 4 .. 64); every lane of the group holds the result
template <int L, class T, class F> __device__ __forceinline__ T group_reduce(T v, F f) {
  if constexpr (L > 1) v = f(v, xor_lane<1>(v));
  if constexpr (L > 2) v = f(v, xor_lane<2>(v));
  if constexpr (L > 4) v = f(v, xor_lane<4>(v));
  if constexpr (L > 8) v = f(v, xor_lane<8>(v));
  if constexpr (L > 16) v = f(v, xor_lane<16>(v));
  if constexpr (L > 32) v = f(v, xor_lane<32>(v));
  return v;
}

}  // namespace ops
}  // namespace tg
