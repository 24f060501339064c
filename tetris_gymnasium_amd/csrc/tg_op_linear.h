// tg_linear_i8: 8-bit rows times 8-bit weights on the integer matrix units, scaled in float32.
//
// acc[m][n] = sum_k x[m][k] w[n][k] in i32 is exact for K <= 65536.  The matrix instructions take signed bytes: u8 rows go in as
// x - 128 (one xor of the top bits), and 128 * sum_k w[n][k] comes back through the accumulator.  The weights are the instruction's
// FIRST operand and the rows its second, so a lane ends up with several columns n of ONE row m; which weight row stands at which
// place of the fragment is free, and it is chosen such that these columns are consecutive: the output leaves in 16-byte stores.
#pragma once
#include "tg_op_common.h"

namespace tg {
namespace ops {

struct LinearArgs {
  const uint8_t* x;
  const int8_t* w;
  const float* ws;
  const float* xs;    // or null
  const float* bias;  // or null
  void* out;
  int64_t rows, k, n, x_stride, w_stride, out_stride;
  int relu;
  int vec;  // 16-byte stores of the output are aligned
};

// 16 bytes of a row starting at byte k, zero behind the row's end (weights: what they hold there decides the sum)
__device__ __forceinline__ v4i load16_row(const uint8_t* row, int64_t k, int64_t K) {
  if (k + 16 <= K) return load16(row + k);
  uint32_t u[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (k + i < K) u[i >> 2] |= (uint32_t)row[k + i] << (8 * (i & 3));
  v4i r = {(int)u[0], (int)u[1], (int)u[2], (int)u[3]};
  return r;
}

// y = act(acc * (xs * ws) + b), rounded once
template <class OT> __device__ __forceinline__ OT linear_out(int acc, float xs, float ws, float b, int relu) {
  float y = fmaf((float)acc, xs * ws, b);
  if (relu) y = y < 0.0f ? 0.0f : y;  // (NaN stays)
  return from_f32<OT>(y);
}

// N consecutive columns of one row, from column n on
template <class OT, int N> __device__ __forceinline__ void linear_store(const LinearArgs& a, int64_t m, int64_t n, const int* acc, float xs) {
  OT* o = (OT*)a.out + m * a.out_stride + n;
  OT y[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t c = n + i < a.n ? n + i : a.n - 1;
    y[i] = linear_out<OT>(acc[i], xs, a.ws[c], a.bias ? a.bias[c] : 0.0f, a.relu);
  }
  if (a.vec && n + N <= a.n) {
#pragma unroll
    for (int i = 0; i < N; i += 16 / (int)sizeof(OT)) {
      v4i v;
      __builtin_memcpy(&v, &y[i], 16);
      *(v4i*)(o + i) = v;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (n + i < a.n) o[i] = y[i];
  }
}

// One wave: 64 columns x 16 rows, the fragments straight from memory.
template <class OT, bool U8> __global__ __launch_bounds__(256) void linear_wave_kernel(const LinearArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.y * 64, m0 = ((int64_t)blockIdx.x * 4 + wave) * 16;
  if (m0 >= a.rows) return;
  const int64_t m = m0 + r < a.rows ? m0 + r : a.rows - 1;
  const uint8_t* xr = a.x + m * a.x_stride;
  const uint8_t* wr[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {  // place (tile t, row 4 p + i) of the fragment holds column 16 p + 4 t + i: lane (q, .) ends with 16 q .. 16 q + 15
    const int64_t n = n0 + 16 * (r >> 2) + 4 * t + (r & 3);
    wr[t] = (const uint8_t*)a.w + (n < a.n ? n : a.n - 1) * a.w_stride;
  }
  v4i acc[4] = {};
  for (int64_t k = 0; k < a.k; k += 64) {
    const int64_t kb = k + 16 * q;
    v4i xf = load16_row(xr, kb, a.k);
    if constexpr (U8) xf ^= (int)0x80808080;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const v4i wf = load16_row(wr[t], kb, a.k);
      if constexpr (U8) {
        const v4i c64 = {0x40404040, 0x40404040, 0x40404040, 0x40404040};
        acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf, c64, acc[t], 0, 0, 0);
        acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf, c64, acc[t], 0, 0, 0);
      }
      acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf, xf, acc[t], 0, 0, 0);
    }
  }
  if (m0 + r < a.rows) {
    int v[16];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[4 * t + i] = acc[t][i];
    linear_store<OT, 16>(a, m, n0 + 16 * q, v, a.xs ? a.xs[m] : 1.0f);
  }
}

}  // namespace ops
}  // namespace tg
