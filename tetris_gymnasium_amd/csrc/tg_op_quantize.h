// tg_quantize_i8: rows of activations to 8-bit integers with one scale each.
//
// s = max(max|x| / 127, 2^-126); q = rint(x / s), half to even, of the REAL quotient.  The quotient is not computed to be rounded
// again: n = rint(x * (1/s)) is the right integer or its neighbour, and x - n s is exact in float32 (one fma: x and n s are
// multiples of one step of s, or of x where x < s, and their difference is below s), so comparing it with s/2 decides, ties too.
// Bound by memory: 2 or 4 bytes in, 1 out per element; a group of LPR lanes holds its row in registers between the maximum and
// the rounding, so each element is read once (rows longer than that are read a second time, from the cache).
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

struct QScale { float s, inv, half; bool ok; };
__device__ __forceinline__ int q_round(float x, const QScale& c) {
  float n = rintf(x * c.inv);
  n = fminf(fmaxf(n, -127.0f), 127.0f);  // (before the check: an overshoot of the estimate at +-127 is undone here)
  const float r = fmaf(-n, c.s, x);      // exact
  const bool odd = ((int)n & 1) != 0;
  if (r > c.half || (r == c.half && odd)) n += 1.0f;
  else if (r < -c.half || (r == -c.half && odd)) n -= 1.0f;
  return c.ok ? (int)n : 0;
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
  uint32_t top = 0;  // max |x| as bits: NaN and infinity compare above every finite value
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t k = ((int64_t)i * LPR + l) * V;
    h[i] = q_load(xr, k < K ? k : K, K);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const uint32_t b = __float_as_uint(to_f32(h[i].v[j])) & 0x7FFFFFFFu;
      top = top > b ? top : b;
    }
  }
  for (int64_t k = ((int64_t)NV * LPR + l) * V; k < K; k += LPR * V) {
    const QVec<T> e = q_load(xr, k, K);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const uint32_t b = __float_as_uint(to_f32(e.v[j])) & 0x7FFFFFFFu;
      top = top > b ? top : b;
    }
  }
  top = group_reduce<(LPR < 64 ? LPR : 64)>(top, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
  if constexpr (LPR > 64) {
    __shared__ uint32_t sh[LPR / 64];
    if ((t & 63) == 0) sh[t >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < LPR / 64; ++i) top = top > sh[i] ? top : sh[i];
  }
  QScale c;
  c.ok = top < 0x7F800000u;
  c.s = fmaxf(__uint_as_float(top) / 127.0f, 0x1p-126f);
  if (!c.ok) c.s = __uint_as_float(0x7FC00000u);
  c.inv = 1.0f / c.s;
  c.half = 0.5f * c.s;
  if (row >= rows) return;
  if (l == 0) scale[row] = c.s;
  int8_t* qr = q + row * qs;
  auto put = [&](int64_t k, const QVec<T>& e) {
    if (k + V <= K) {
      uint32_t w[V / 4];
#pragma unroll
      for (int j = 0; j < V / 4; ++j)
        w[j] = (uint32_t)(q_round(to_f32(e.v[4 * j]), c) & 255) | ((uint32_t)(q_round(to_f32(e.v[4 * j + 1]), c) & 255) << 8) |
               ((uint32_t)(q_round(to_f32(e.v[4 * j + 2]), c) & 255) << 16) | ((uint32_t)(q_round(to_f32(e.v[4 * j + 3]), c) & 255) << 24);
      __builtin_memcpy(qr + k, w, V);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (k + j < K) qr[k + j] = (int8_t)q_round(to_f32(e.v[j]), c);
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
