// tg_quantize_i8: rows of activations to 8-bit integers with one scale each.
//
// s = max(max|x| / 127, 2^-126); q = rint(x / s), half to even, of the REAL quotient.  The quotient is not computed to be rounded
// again: n = rint(x * (1/s)) is the right integer or its neighbour, and x - n s is exact in float32 (one fma: x and n s are
// multiples of one step of s, or of x where x < s, and their difference is below s), so comparing it with s/2 decides, ties too.
// Bound by memory: 2 or 4 bytes in, 1 out per element; a group of LPR lanes holds its row in registers between the maximum and
// the rounding, so each element is read once (rows longer than that are read a second time, from the cache).  65 536 x 256 bf16 (50 MB):
// 10.8 us = 4.7 TB/s, 8 192 x 4 096: 18.5 us = 5.5 TB/s, 655 360 x 32: 13.7 us (sixteen lanes a row, most of them idle: 38).
#pragma once
#include "tg_op_common.h"

namespace tg {
namespace ops {

template <class T> constexpr int kQVec = 16 / (int)sizeof(T);  // elements of one 16-byte load

template <class T> struct QVec { T v[kQVec<T>]; };

// elements k .. k + 15/sizeof(T) of a row of K (zero behind its end)
template <class T> __device__ __forceinline__ QVec<T> q_load(const T* row, int64_t k, int64_t K) {
  QVec<T> r;
  if (k + kQVec<T> <= K) {
    const v4i u = load16(row + k);
    __builtin_memcpy(&r, &u, 16);
  } else {
#pragma unroll
    for (int i = 0; i < kQVec<T>; ++i) {
      T z{};
      r.v[i] = z;
      if (k + i < K) r.v[i] = row[k + i];
    }
  }
  return r;
}

struct QScale { float s, inv, half; };
// exactly: the neighbour decided by the remainder, halves to even
__device__ __forceinline__ uint32_t q_exact(float x, const QScale& c) {
  float n = rintf(x * c.inv);
  n = fminf(fmaxf(n, -127.0f), 127.0f);  // (before the check: an overshoot of the estimate at +-127 is undone here)
  const float r = fmaf(-n, c.s, x);      // exact
  const bool odd = ((int)n & 1) != 0;
  if (r > c.half || (r == c.half && odd)) n += 1.0f;
  else if (r < -c.half || (r == -c.half && odd)) n -= 1.0f;
  return (uint32_t)(int)n & 255u;
}
// Four at a time: with 1.5 * 2^23 added the estimate lies in the low byte of the float's bits, and it is right wherever the remainder
// is below half a step — almost always; the rest of the wave's vector goes the exact way.
__device__ __forceinline__ uint32_t q_round4(const float (&x)[4], const QScale& c) {
  const float magic = 12582912.0f;
  float y[4];
  bool close = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    y[i] = fmaf(x[i], c.inv, magic);
    close |= !(fabsf(fmaf(-(y[i] - magic), c.s, x[i])) < c.half);
  }
  if (__builtin_expect(__ballot(close) != 0, 0)) return q_exact(x[0], c) | (q_exact(x[1], c) << 8) | (q_exact(x[2], c) << 16) | (q_exact(x[3], c) << 24);
  const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(y[1]), __float_as_uint(y[0]), 0x0C0C0400u);
  const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(y[3]), __float_as_uint(y[2]), 0x04000C0Cu);
  return lo | hi;
}

// the largest |x| of a vector, as bits of the type (NaN and infinity compare above every finite value), joined with `top`
template <class T> __device__ __forceinline__ uint32_t q_top(const QVec<T>& e, uint32_t top) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t b = __float_as_uint(e.v[j]) & 0x7FFFFFFFu;
      top = top > b ? top : b;
    }
  } else {  // two 16-bit maxima side by side
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    uint32_t w[4];
    __builtin_memcpy(w, &e, 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t b = w[j] & 0x7FFF7FFFu;
      u16x2 p, q;
      __builtin_memcpy(&p, &b, 4);
      __builtin_memcpy(&q, &top, 4);
      const u16x2 m = __builtin_elementwise_max(p, q);
      __builtin_memcpy(&top, &m, 4);
    }
  }
  return top;
}
// ... its value; NaN or infinity where the row holds one
template <class T> __device__ __forceinline__ float q_top_value(uint32_t top) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(top);
  else {
    const uint16_t b = (uint16_t)((top >> 16) > (top & 0xFFFFu) ? top >> 16 : top);
    T v;
    __builtin_memcpy(&v, &b, 2);
    return to_f32(v);
  }
}
template <class T> __device__ __forceinline__ uint32_t q_top_join(uint32_t a, uint32_t b) {
  if constexpr (sizeof(T) == 4) return a > b ? a : b;
  else {
    const uint32_t lo = (a & 0xFFFFu) > (b & 0xFFFFu) ? a & 0xFFFFu : b & 0xFFFFu, hi = (a >> 16) > (b >> 16) ? a >> 16 : b >> 16;
    return lo | (hi << 16);
  }
}

// LPR lanes per row (16, 64: rows share a wave / a row each; 256: a workgroup a row), NV loads held per lane
template <class T, int LPR, int NV> __global__ __launch_bounds__(256) void quantize_kernel(const T* __restrict__ x, int64_t rows, int64_t K,
                                                                                         int64_t xs, int8_t* __restrict__ q, int64_t qs,
                                                                                         float* __restrict__ scale) {
  constexpr int V = kQVec<T>, RPB = 256 / LPR;
  const int t = threadIdx.x, l = t % LPR;
  const int64_t row = (int64_t)blockIdx.x * RPB + t / LPR;
  const int64_t rr = row < rows ? row : rows - 1;  // (lanes of a row beyond the last repeat it and store nothing)
  const T* xr = x + rr * xs;
  QVec<T> h[NV];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t k = ((int64_t)i * LPR + l) * V;
    if (k < K) h[i] = q_load(xr, k, K);
    else h[i] = QVec<T>{};
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) top = q_top<T>(h[i], top);
  for (int64_t k = ((int64_t)NV * LPR + l) * V; k < K; k += LPR * V) top = q_top<T>(q_load(xr, k, K), top);
  top = group_reduce<(LPR < 64 ? LPR : 64)>(top, q_top_join<T>);
  if constexpr (LPR > 64) {
    __shared__ uint32_t sh[LPR / 64];
    if ((t & 63) == 0) sh[t >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < LPR / 64; ++i) top = q_top_join<T>(top, sh[i]);
  }
  const float most = q_top_value<T>(top);
  const bool ok = most < __builtin_inff();
  QScale c;
  c.s = ok ? fmaxf(most / 127.0f, 0x1p-126f) : __uint_as_float(0x7FC00000u);
  c.inv = ok ? 1.0f / c.s : 0.0f;
  c.half = 0.5f * c.s;
  if (row >= rows) return;
  if (l == 0) scale[row] = c.s;
  int8_t* qr = q + row * qs;
  auto put = [&](int64_t k, const QVec<T>& e) {
    uint32_t w[V / 4];
#pragma unroll
    for (int j = 0; j < V / 4; ++j) {
      const float x[4] = {to_f32(e.v[4 * j]), to_f32(e.v[4 * j + 1]), to_f32(e.v[4 * j + 2]), to_f32(e.v[4 * j + 3])};
      w[j] = q_round4(x, c);
      w[j] = ok ? w[j] : 0;
    }
    if (k + V <= K) {
      __builtin_memcpy(qr + k, w, V);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (k + j < K) qr[k + j] = (int8_t)(w[j / 4] >> (8 * (j % 4)));
    }
  };
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t k = ((int64_t)i * LPR + l) * V;
    if (k < K) put(k, h[i]);
  }
  for (int64_t k = ((int64_t)NV * LPR + l) * V; k < K; k += LPR * V) put(k, q_load(xr, k, K));
}

}  // namespace ops
}  // namespace tg
