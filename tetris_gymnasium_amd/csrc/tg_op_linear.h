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
template <class OT, int N> __device__ __forceinline__ void linear_put(const LinearArgs& a, int64_t m, int64_t n, const OT (&y)[N]) {
  OT* o = (OT*)a.out + m * a.out_stride + n;
  constexpr int V = 16 / (int)sizeof(OT) < N ? 16 / (int)sizeof(OT) : N;
  if (n + N <= a.n) {  // (vector stores at any address: rows of an odd width start anywhere)
#pragma unroll
    for (int i = 0; i < N; i += V) {
      struct __attribute__((packed, aligned(1))) { OT e[V]; } v;
#pragma unroll
      for (int j = 0; j < V; ++j) v.e[j] = y[i + j];
      __builtin_memcpy((void*)(o + i), &v, sizeof(v));
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (n + i < a.n) o[i] = y[i];
  }
}
template <class OT, int N> __device__ __forceinline__ void linear_store(const LinearArgs& a, int64_t m, int64_t n, const int (&acc)[N], float xs) {
  OT y[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t c = n + i < a.n ? n + i : a.n - 1;
    y[i] = linear_out<OT>(acc[i], xs, a.ws[c], a.bias ? a.bias[c] : 0.0f, a.relu);
  }
  linear_put<OT, N>(a, m, n, y);
}

// ---- short rows (K <= 64 * KS), many of them ------------------------------------------------------------------------------------
// Bound by memory: a byte of input is used N times, N <= a few hundred.  A wave keeps the weights of 64 columns in registers (16 KS
// of them) and walks over tiles of 16 rows, the next tile's fragments in flight behind the present one's products.
template <class OT, bool U8, int KS> __global__ __launch_bounds__(256) void linear_rows_kernel(const LinearArgs a, int strips) {
  // C columns make 16 bytes of output, G tiles a lane's C columns: the four lanes of a row then store 64 bytes side by side at a time
  constexpr int C = 16 / (int)sizeof(OT), G = C / 4;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  const int64_t n0 = ((int64_t)blockIdx.y * strips + wave % strips) * 64;  // `strips` of the four waves side by side, the others below
  const int below = 4 / strips;
  const int64_t tiles = (a.rows + 15) / 16, step = (int64_t)gridDim.x * below;
  int64_t tile = (int64_t)blockIdx.x * below + wave / strips;
  if (n0 >= a.n || tile >= tiles) return;
  const uint8_t* const last = a.x + (a.rows - 1) * a.x_stride + a.k - 16;  // the last address that 16 bytes may be read from
  auto fetch = [&](int64_t t, v4i* f) {
    const int64_t m = t * 16 + r < a.rows ? t * 16 + r : a.rows - 1;
    const uint8_t* xr = a.x + m * a.x_stride;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int kb = 64 * s + 16 * q;
      v4i v = {0, 0, 0, 0};
      if (kb < a.k) {  // (bytes behind the row's end meet weights of zero)
        if (xr + kb <= last) v = load16(xr + kb);
        else v = load16_row(xr, kb, a.k);
      }
      f[s] = v;
    }
  };
  v4i w[KS][4], init[4] = {}, f[KS];
  fetch(tile, f);
#pragma unroll
  for (int t = 0; t < 4; ++t) {  // place (tile t, row 4 p + i) of the fragment holds column 4 C (t / G) + C p + 4 (t % G) + i: see C
    const int64_t n = n0 + 4 * C * (t / G) + C * (r >> 2) + 4 * (t % G) + (r & 3);
    const uint8_t* wr = (const uint8_t*)a.w + (n < a.n ? n : a.n - 1) * a.w_stride;
#pragma unroll
    for (int s = 0; s < KS; ++s) w[s][t] = load16_row(wr, 64 * s + 16 * q, a.k);
  }
  if constexpr (U8) {
    const v4i c64 = {0x40404040, 0x40404040, 0x40404040, 0x40404040};  // 64 + 64 times the weights: what x - 128 lacks
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        init[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[s][t], c64, init[t], 0, 0, 0);
        init[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[s][t], c64, init[t], 0, 0, 0);
      }
  }
  float ws[16], b[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    int64_t c = n0 + 4 * C * (i / C) + C * q + i % C;
    c = c < a.n ? c : a.n - 1;
    ws[i] = a.ws[c];
    b[i] = a.bias ? a.bias[c] : 0.0f;
  }
  while (true) {
    const int64_t next = tile + step;
    v4i g[KS];
    if (next < tiles) fetch(next, g);
    const int64_t m = tile * 16 + r;
    float xs = 1.0f;
    if (a.xs && m < a.rows) xs = a.xs[m];
    v4i acc[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[t] = init[t];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      if constexpr (U8) f[s] ^= (int)0x80808080;
#pragma unroll
      for (int t = 0; t < 4; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[s][t], f[s], acc[t], 0, 0, 0);
    }
    if (m < a.rows) {
#pragma unroll
      for (int j = 0; j < 16; j += C) {
        OT y[C];
#pragma unroll
        for (int i = 0; i < C; ++i) y[i] = linear_out<OT>(acc[(i + j) >> 2][(i + j) & 3], xs, ws[i + j], b[i + j], a.relu);
        linear_put<OT, C>(a, m, n0 + 4 * j + C * q, y);
      }
    }
    if (next >= tiles) return;
    tile = next;
#pragma unroll
    for (int s = 0; s < KS; ++s) f[s] = g[s];
  }
}

// ---- few rows (<= 16 * U), any K -------------------------------------------------------------------------------------------------
// Bound by reading the weights once: a workgroup takes 16 T columns and its waves share K, each summing its part; the parts are added
// through LDS (integers: in any order the same).
template <class OT, bool U8, int T, int U> __global__ __launch_bounds__(512) void linear_few_kernel(const LinearArgs a, int kw) {
  __shared__ v4i part[7][T * U][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, r = lane & 15, q = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * (16 * T), m0 = (int64_t)blockIdx.y * (16 * U);
  const int64_t k0 = (int64_t)wave * kw, k1 = k0 + kw < a.k ? k0 + kw : a.k;  // (kw is a multiple of 64)
  const uint8_t *xr[U], *wr[T];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t m = m0 + 16 * u + r;
    xr[u] = a.x + (m < a.rows ? m : a.rows - 1) * a.x_stride;
  }
#pragma unroll
  for (int t = 0; t < T; ++t) {  // place (t, 4 p + i) holds column 4 T p + 4 t + i: lane (q, .) ends with 4 T consecutive ones
    const int64_t n = n0 + 4 * T * (r >> 2) + 4 * t + (r & 3);
    wr[t] = (const uint8_t*)a.w + (n < a.n ? n : a.n - 1) * a.w_stride;
  }
  v4i acc[T][U] = {};
  auto product = [&](const v4i (&wf)[T], v4i (&xf)[U]) {
    const v4i c64 = {0x40404040, 0x40404040, 0x40404040, 0x40404040};
#pragma unroll
    for (int u = 0; u < U; ++u)
      if constexpr (U8) xf[u] ^= (int)0x80808080;
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if constexpr (U8) {
          acc[t][u] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[t], c64, acc[t][u], 0, 0, 0);
          acc[t][u] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[t], c64, acc[t][u], 0, 0, 0);
        }
        acc[t][u] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[t], xf[u], acc[t][u], 0, 0, 0);
      }
  };
  int64_t k = k0;
  constexpr int UN = 4;  // k-steps whose loads are in flight together
  for (; k + 64 * UN <= k1; k += 64 * UN) {
    v4i wf[UN][T], xf[UN][U];
#pragma unroll
    for (int i = 0; i < UN; ++i) {
#pragma unroll
      for (int t = 0; t < T; ++t) wf[i][t] = load16(wr[t] + k + 64 * i + 16 * q);
#pragma unroll
      for (int u = 0; u < U; ++u) xf[i][u] = load16(xr[u] + k + 64 * i + 16 * q);
    }
#pragma unroll
    for (int i = 0; i < UN; ++i) product(wf[i], xf[i]);
  }
  for (; k < k1; k += 64) {
    v4i wf[T], xf[U];
#pragma unroll
    for (int t = 0; t < T; ++t) wf[t] = load16_row(wr[t], k + 16 * q, a.k);
#pragma unroll
    for (int u = 0; u < U; ++u) xf[u] = load16_row(xr[u], k + 16 * q, a.k);
    product(wf, xf);
  }
  if (wave) {
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int u = 0; u < U; ++u) part[wave - 1][t * U + u][lane] = acc[t][u];
  }
  __syncthreads();
  if (wave) return;
  for (int o = 1; o < waves; ++o)
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int u = 0; u < U; ++u) acc[t][u] += part[o - 1][t * U + u][lane];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t m = m0 + 16 * u + r;
    if (m < a.rows) {
      int v[4 * T];
#pragma unroll
      for (int i = 0; i < 4 * T; ++i) v[i] = acc[i >> 2][u][i & 3];
      linear_store<OT, 4 * T>(a, m, n0 + 4 * T * q, v, a.xs ? a.xs[m] : 1.0f);
    }
  }
}

// ---- everything else: tiles of BM rows x BN columns through LDS -------------------------------------------------------------------
// 128 bytes of K at a time, two buffers: while one is multiplied the next one arrives.  Sixteen bytes (row, c) lie at place c ^ (row >> 1
// & 7) of their row, so the sixteen lanes that read one column of chunks together hit all banks once.  ALIGNED (16-byte addresses
// throughout): the tiles go from memory to LDS without passing registers.  32 x 32 x 32 products; the LDS row d of the weights holds
// column 16 (d >> 2 & 1) + 4 (d >> 3) + (d & 3) of its 32, so that a lane ends with sixteen consecutive columns of one row.
__device__ const v4i kZero16 = {0, 0, 0, 0};

template <class OT, bool U8, int BM, int BN, int WM, int WN, bool ALIGNED>
__global__ __launch_bounds__(WM * WN * 64) void linear_tile_kernel(const LinearArgs a, int mt, int nt) {
  constexpr int THREADS = WM * WN * 64, BK = 128, MT = BM / WM / 32, NT = BN / WN / 32;
  constexpr int LOADS = (BM + BN) * 8 / THREADS;  // 16-byte chunks of a stage per thread
  static_assert((BM + BN) * 8 % THREADS == 0 && BM * 8 % THREADS == 0, "whole waves per operand");
  extern __shared__ uint8_t lds[];  // [2][(BM + BN) * BK]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave / WN, wn = wave % WN;
  // workgroups go to the eight dies in turn: each die gets a contiguous run of tiles, in columns of eight row tiles (their operands
  // stay in its cache)
  int id = blockIdx.x;
  const int total = mt * nt;
  {
    const int per = total / 8, rest = total % 8, die = id % 8, i = id / 8;
    id = die * per + (die < rest ? die : rest) + i;
  }
  constexpr int GROUP = 8;
  const int band = id / (GROUP * nt), in = id % (GROUP * nt), high = mt - band * GROUP < GROUP ? mt - band * GROUP : GROUP;
  const int64_t m0 = (int64_t)(band * GROUP + in % high) * BM, n0 = (int64_t)(in / high) * BN;

  const uint8_t* src[LOADS];
  int kin[LOADS];  // byte of the row the chunk starts at, in the stage
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int c = i * THREADS + tid, row = c >> 3;  // place c of the stage: X rows, then W rows
    kin[i] = ((c & 7) ^ ((row >> 1) & 7)) * 16;
    if (i * THREADS < BM * 8) {
      const int64_t m = m0 + row;
      src[i] = a.x + (m < a.rows ? m : a.rows - 1) * a.x_stride;
    } else {
      const int d = row - BM;
      const int64_t n = n0 + (d & ~31) + 16 * ((d >> 2) & 1) + 4 * ((d >> 3) & 3) + (d & 3);
      src[i] = (const uint8_t*)a.w + (n < a.n ? n : a.n - 1) * a.w_stride;
    }
    src[i] += kin[i];
  }
  const int64_t steps = (a.k + BK - 1) / BK;
  v4i hold[ALIGNED ? 1 : LOADS];
  auto load = [&](int64_t s, uint8_t* stage) {
    const int64_t k = s * BK;
    if constexpr (ALIGNED) {
      const bool whole = k + BK <= a.k;
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const uint8_t* p = src[i] + k;
        if (!whole && k + kin[i] >= a.k) p = (const uint8_t*)&kZero16;
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)p,
                                         (__attribute__((address_space(3))) void*)(stage + (i * THREADS + wave * 64) * 16), 16, 0, 0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) hold[i] = load16_row(src[i] - kin[i], k + kin[i], a.k);
    }
  };
  auto settle = [&](uint8_t* stage) {
    if constexpr (ALIGNED) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    } else {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) *(v4i*)(stage + (i * THREADS + tid) * 16) = hold[i];
    }
  };
  v16i acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
  int sum[NT] = {};  // U8: of the weights of the lane's fragment row
  const int lr = lane & 31, half = lane >> 5, sw = (lr >> 1) & 7;
  constexpr int STAGE = (BM + BN) * BK;
  if (steps > 0) load(0, lds);
  for (int64_t s = 0; s < steps; ++s) {
    uint8_t* here = lds + (s & 1) * STAGE;
    settle(here);
    __syncthreads();  // this stage is complete, and nobody reads the other one any more
    if (s + 1 < steps) load(s + 1, lds + ((s + 1) & 1) * STAGE);
    const uint8_t* xb = here + (wm * (BM / WM) + lr) * BK;
    const uint8_t* wb = here + (BM + wn * (BN / WN) + lr) * BK;
#pragma unroll
    for (int kk = 0; kk < BK / 32; ++kk) {
      const int at = ((kk * 2 + half) ^ sw) * 16;
      v4i xf[MT], wf[NT];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        xf[i] = *(const v4i*)(xb + i * 32 * BK + at);
        if constexpr (U8) xf[i] ^= (int)0x80808080;
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        wf[j] = *(const v4i*)(wb + j * 32 * BK + at);
        if constexpr (U8) {
#pragma unroll
          for (int e = 0; e < 4; ++e) sum[j] = __builtin_amdgcn_sdot4(wf[j][e], 0x01010101, sum[j], false);
        }
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[j], xf[i], acc[i][j], 0, 0, 0);
    }
  }
  // the 128 sum_k w that x - 128 lacks, from the lane that holds column d of the fragment to those that hold its results
  int lack[NT][16];
  if constexpr (U8) {
    __syncthreads();
    int* sh = (int*)lds + wave * (NT * 32);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int all = sum[j] + (int)xor_lane<32>((uint32_t)sum[j]);
      if (half == 0) sh[j * 32 + 16 * ((lr >> 2) & 1) + 4 * (lr >> 3) + (lr & 3)] = all << 7;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) lack[j][e] = sh[j * 32 + half * 16 + e];
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int64_t n = n0 + wn * (BN / WN) + j * 32 + half * 16;
    float ws[16], b[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int64_t c = n + e < a.n ? n + e : a.n - 1;
      ws[e] = a.ws[c];
      b[e] = a.bias ? a.bias[c] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int64_t m = m0 + wm * (BM / WM) + i * 32 + lr;
      if (m < a.rows) {
        const float xs = a.xs ? a.xs[m] : 1.0f;
        OT y[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          int v = acc[i][j][e];
          if constexpr (U8) v += lack[j][e];
          y[e] = linear_out<OT>(v, xs, ws[e], b[e], a.relu);
        }
        linear_put<OT, 16>(a, m, n, y);
      }
    }
  }
}

}  // namespace ops
}  // namespace tg
