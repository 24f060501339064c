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

// The bytes of an operand: reads of 16 bytes stay inside [begin, end).
struct Span { const uint8_t *begin, *end; };
__device__ __forceinline__ Span x_span(const LinearArgs& a) { return {a.x, a.x + (a.rows - 1) * a.x_stride + a.k}; }
__device__ __forceinline__ Span w_span(const LinearArgs& a) { return {(const uint8_t*)a.w, (const uint8_t*)a.w + (a.n - 1) * a.w_stride + a.k}; }

// N times the 16 bytes at p[i], wherever they lie; what is behind the operand's end reads as zero.  Loads near the end move in front of
// it and are shifted down afterwards, so that none of the N waits for another; an operand below 16 bytes is read byte by byte.
template <int N> __device__ __forceinline__ void load16_inside(const uint8_t* const (&p)[N], const Span& o, v4i (&v)[N]) {
  if (o.end - o.begin >= 16) {
    const uint8_t* const last = o.end - 16;
    int64_t over[N];
    bool any = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint8_t* q = p[i] < last ? p[i] : last;
      v[i] = load16(q);
      over[i] = p[i] - q;
      any |= over[i] > 0;
    }
    if (__ballot(any)) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        unsigned __int128 u;
        __builtin_memcpy(&u, &v[i], 16);
        u = over[i] < 16 ? u >> (8 * (int)over[i]) : 0;
        __builtin_memcpy(&v[i], &u, 16);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      unsigned __int128 u = 0;
#pragma unroll 1
      for (int j = 15; j >= 0; --j) u = (u << 8) | (p[i] + j < o.end ? p[i][j] : 0);
      __builtin_memcpy(&v[i], &u, 16);
    }
  }
}
// the first n of 16 bytes (weights: behind the row's end they have to be zero, what the rows hold there then does not count)
__device__ __forceinline__ v4i first_bytes(v4i v, int n) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int b = n - 4 * j;
    v[j] &= b >= 4 ? -1 : b <= 0 ? 0 : (1 << (8 * b)) - 1;
  }
  return v;
}

// y = act(acc * (xs * ws) + b), rounded once
template <class OT> __device__ __forceinline__ OT linear_out(int acc, float xs, float ws, float b, int relu) {
  float y = fmaf((float)acc, xs * ws, b);
  if (relu) y = y < 0.0f ? 0.0f : y;  // (NaN stays)
  return from_f32<OT>(y);
}

// N consecutive columns of one row, from column n on
template <class OT, int N> __device__ __forceinline__ void linear_put(const LinearArgs& a, int64_t m, int64_t n, const OT (&y)[N], bool wide = false) {
  OT* o = (OT*)a.out + m * a.out_stride + n;
  constexpr int V = 16 / (int)sizeof(OT) < N ? 16 / (int)sizeof(OT) : N;
  if (wide || n + N <= a.n) {  // (vector stores at any address: rows of an odd width start anywhere)
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
// of them) and walks over tiles of 16 rows, the next tile's fragments in flight behind the present one's products.  65 536 boards of
// 200 bytes into 256 bf16 (47 MB): 16.3 us = 2.9 TB/s, 7.7 of them until the first tile is out; without its stores 12, without
// loads and stores 11: 2 023 vector instructions a wave at two waves a SIMD are 6 - 7 us of issue.  Two or three tiles in flight, or three workgroups per unit, are not faster.
template <class OT, bool U8, int KS> __global__ __launch_bounds__(256) void linear_rows_kernel(const LinearArgs a, int shift, int64_t inside) {
  // C columns make 16 bytes of output, G tiles a lane's C columns: the four lanes of a row then store 64 bytes side by side at a time
  constexpr int C = 16 / (int)sizeof(OT), G = C / 4;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  const int64_t n0 = ((int64_t)((blockIdx.y << shift) + (wave & ((1 << shift) - 1)))) * 64;  // 2^shift of the four waves side by side, the others below
  const int below = 4 >> shift;
  const int64_t tiles = (a.rows + 15) / 16, step = (int64_t)gridDim.x * below;
  int64_t tile = (int64_t)blockIdx.x * below + __builtin_amdgcn_readfirstlane(wave >> shift);
  if (n0 >= a.n || tile >= tiles) return;
  const Span xo = x_span(a);
  // (tiles below `inside` read inside the operand with all their loads; bytes behind a row's end meet weights of zero)
  auto fetch = [&](int64_t t, v4i (&f)[KS]) {
    const uint8_t* xr = a.x + (t * 16 + r) * a.x_stride + 16 * q;
    if (t < inside) {
#pragma unroll
      for (int s = 0; s < KS; ++s) f[s] = load16(xr + 64 * s);
    } else {
      const uint8_t* p[KS];
#pragma unroll
      for (int s = 0; s < KS; ++s) p[s] = xr + 64 * s;
      load16_inside<KS>(p, xo, f);
    }
  };
  v4i w[4][KS], init[4] = {}, f[KS];
  fetch(tile, f);
  const Span wo = w_span(a);
#pragma unroll
  for (int t = 0; t < 4; ++t) {  // place (tile t, row 4 p + i) of the fragment holds column 4 C (t / G) + C p + 4 (t % G) + i: see C
    const int64_t n = n0 + 4 * C * (t / G) + C * (r >> 2) + 4 * (t % G) + (r & 3);
    const uint8_t* p[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) p[s] = (const uint8_t*)a.w + (n < a.n ? n : a.n - 1) * a.w_stride + 64 * s + 16 * q;
    load16_inside<KS>(p, wo, w[t]);
  }
  const bool wide = n0 + 64 <= a.n;
  struct alignas(8) Column { float ws, b; };
  __shared__ Column column[4][64];  // of each wave's strip: 32 registers less (up to K = 128 a third wave per SIMD; above, 180 - 200: two)
  {
    const int64_t c = n0 + lane < a.n ? n0 + lane : a.n - 1;
    column[wave][lane] = {a.ws[c], a.bias ? a.bias[c] : 0.0f};
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      w[t][s] = first_bytes(w[t][s], (int)a.k - 64 * s - 16 * q);
      if constexpr (U8) {
        const v4i c64 = {0x40404040, 0x40404040, 0x40404040, 0x40404040};  // 64 + 64 times the weights: what x - 128 lacks
        init[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[t][s], c64, init[t], 0, 0, 0);
        init[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[t][s], c64, init[t], 0, 0, 0);
      }
    }
  while (true) {
    const int64_t next = tile + step, m = tile * 16 + r;
    v4i g[KS];
    if (next < tiles) fetch(next, g);
    float xs = 1.0f;
    if (a.xs) xs = a.xs[m < a.rows ? m : a.rows - 1];
    v4i acc[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[t] = init[t];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      if constexpr (U8) f[s] ^= (int)0x80808080;
#pragma unroll
      for (int t = 0; t < 4; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[t][s], f[s], acc[t], 0, 0, 0);
    }
    float y[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const Column c = column[wave][4 * C * (i / C) + C * q + i % C];
      y[i] = fmaf((float)acc[i >> 2][i & 3], xs * c.ws, c.b);
    }
    if (a.relu) {
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] = y[i] < 0.0f ? 0.0f : y[i];
    }
    if (m < a.rows) {
#pragma unroll
      for (int j = 0; j < 16; j += C) {
        OT o[C];
#pragma unroll
        for (int i = 0; i < C; ++i) o[i] = from_f32<OT>(y[i + j]);
        linear_put<OT, C>(a, m, n0 + 4 * j + C * q, o, wide);
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
// through LDS (integers: in any order the same).  8 x 4 096 -> 8 192 (34 MB): 8.3 us = 4.1 TB/s; one board of 200 bytes -> 256: 3.7 us.
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
    const uint8_t *pw[T], *px[U];
#pragma unroll
    for (int t = 0; t < T; ++t) pw[t] = wr[t] + k + 16 * q;
#pragma unroll
    for (int u = 0; u < U; ++u) px[u] = xr[u] + k + 16 * q;
    load16_inside<T>(pw, w_span(a), wf);
    load16_inside<U>(px, x_span(a), xf);
#pragma unroll
    for (int t = 0; t < T; ++t) wf[t] = first_bytes(wf[t], (int)(a.k - k) - 16 * q);
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
// 128 bytes of K at a time in two buffers: one arrives while the other is multiplied.  Sixteen bytes (row, c) lie at place
// c ^ (row >> 1 & 7) of their row, so the sixteen lanes that read one column of chunks together hit all banks once (no conflict
// counted).  ALIGNED (16-byte addresses throughout): the tiles go from memory to LDS without passing registers.  32 x 32 x 32 products;
// the LDS row d of the weights holds column 16 (d >> 2 & 1) + 4 (d >> 3) + (d & 3) of its 32, so that a lane ends with sixteen consecutive
// columns of one row.
// Bound by the matrix units' power: 8 192 x 4 096 x 4 096 with random bytes runs at 1.67 - 2.02 POP/s (156 - 164 us at the median, 136 at best), the
// products alone, without loads, LDS reads and barriers, at 2.2 - 2.6, and the same kernel on zeros at 2.3.  64 bytes of K in three to five stages were
// slower (150 - 168 us: half lines), tiles of 256 x 128 and 128 x 128 too (165, 162 us: more loads), four waves of 128 x 128 too (167 us).
__device__ const v4i kZero16 = {0, 0, 0, 0};

template <class OT, bool U8, int BM, int BN, int WM, int WN, bool ALIGNED>
__global__ __launch_bounds__(WM * WN * 64) void linear_tile_kernel(const LinearArgs a, int mt, int nt) {
  constexpr int THREADS = WM * WN * 64, MT = BM / WM / 32, NT = BN / WN / 32;
  constexpr int BK = 128, CH = BK / 16, LOADS = (BM + BN) * CH / THREADS;  // 16-byte chunks of a row, of a stage per thread
  static_assert((BM + BN) * CH % THREADS == 0 && BM * CH % THREADS == 0, "whole waves per operand");
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
    const int c = i * THREADS + tid, row = c / CH;  // place c of the stage: X rows, then W rows
    kin[i] = ((c % CH) ^ ((row >> 1) % CH)) * 16;
    if (i * THREADS < BM * CH) {
      const int64_t m = m0 + row;
      src[i] = a.x + (m < a.rows ? m : a.rows - 1) * a.x_stride;
    } else {
      const int d = row - BM;
      const int64_t n = n0 + (d & ~31) + 16 * ((d >> 2) & 1) + 4 * ((d >> 3) & 3) + (d & 3);
      src[i] = (const uint8_t*)a.w + (n < a.n ? n : a.n - 1) * a.w_stride;
    }
    if constexpr (ALIGNED) src[i] += kin[i];
  }
  const int steps = (int)((a.k + BK - 1) / BK);
  constexpr int STAGE = (BM + BN) * BK;
  v4i hold[ALIGNED ? 1 : LOADS];
  auto load = [&](int s) {
    const int64_t k = (int64_t)s * BK;
    if constexpr (ALIGNED) {
      uint8_t* stage = lds + (s & 1) * STAGE;
      const bool whole = k + BK <= a.k;
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const uint8_t* p = src[i] + k;
        if (!whole && k + kin[i] >= a.k) p = (const uint8_t*)&kZero16;
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)p,
                                         (__attribute__((address_space(3))) void*)(stage + (i * THREADS + wave * 64) * 16), 16, 0, 0);
      }
    } else {
      constexpr int XL = BM * CH / THREADS;  // the first of them are of X
      const uint8_t *px[XL], *pw[LOADS - XL];
      v4i vx[XL], vw[LOADS - XL];
#pragma unroll
      for (int i = 0; i < LOADS; ++i) (i < XL ? px[i < XL ? i : 0] : pw[i < XL ? 0 : i - XL]) = src[i] + k + kin[i];
      load16_inside<XL>(px, x_span(a), vx);
      load16_inside<LOADS - XL>(pw, w_span(a), vw);
#pragma unroll
      for (int i = 0; i < LOADS; ++i) hold[i] = i < XL ? vx[i < XL ? i : 0] : first_bytes(vw[i < XL ? 0 : i - XL], (int)(a.k - k) - kin[i]);
    }
  };
  auto settle = [&](int s) {  // stage s of this wave has arrived
    if constexpr (ALIGNED) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    } else {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) *(v4i*)(lds + (s & 1) * STAGE + (i * THREADS + tid) * 16) = hold[i];
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
  const int lr = lane & 31, half = lane >> 5, sw = (lr >> 1) % CH;
  constexpr int KK = BK / 32;
  v4i xf[2][MT], wf[2][NT];
  auto read = [&](int s, int kk, int f) {  // the fragments of 32 bytes of K
    const uint8_t* here = lds + (s & 1) * STAGE;
    const int at = ((kk * 2 + half) ^ sw) * 16;
#pragma unroll
    for (int j = 0; j < NT; ++j) wf[f][j] = *(const v4i*)(here + (BM + wn * (BN / WN) + j * 32 + lr) * BK + at);
#pragma unroll
    for (int i = 0; i < MT; ++i) xf[f][i] = *(const v4i*)(here + (wm * (BM / WM) + i * 32 + lr) * BK + at);
  };
  auto multiply = [&](int f) {
    if constexpr (U8) {
#pragma unroll
      for (int i = 0; i < MT; ++i) xf[f][i] ^= (int)0x80808080;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[j] = __builtin_amdgcn_sdot4(wf[f][j][e], 0x01010101, sum[j], false);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[f][j], xf[f][i], acc[i][j], 0, 0, 0);
  };
  auto interleave = [] {  // a read of the next fragments behind each of the first products
    if constexpr (MT * NT >= MT + NT) {
#pragma unroll
      for (int i = 0; i < MT + NT; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, MT * NT - MT - NT, 0);
    }
  };
  auto meet = [&] {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
  };
  if (steps > 0) {
    load(0);
    settle(0);
    meet();
    if (steps > 1) load(1);
    read(0, 0, 0);
  }
  for (int s = 0; s < steps; ++s) {
#pragma unroll
    for (int kk = 0; kk + 1 < KK; ++kk) {
      read(s, kk + 1, (kk + 1) & 1);
      multiply(kk & 1);
      interleave();
    }
    if (s + 1 < steps) {  // everything of this stage is in registers: meet, refill its buffer, and start on the next one
      settle(s + 1);
      meet();
      if (s + 2 < steps) load(s + 2);
      read(s + 1, 0, 0);
    }
    multiply((KK - 1) & 1);
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
  // The results leave through the wave's own piece of LDS, so that they are stored in rows of BN / WN columns: a lane's sixteen columns
  // alone would be pieces of 16 bytes all over the lines (a 256 x 256 tile in bf16 took 15 us with its setup, 13 us like this).
  float ws[NT][16], b[NT][16];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int64_t n = n0 + wn * (BN / WN) + j * 32 + half * 16;
    if (n + 16 <= a.n) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        ws[j][e] = a.ws[n + e];
        b[j][e] = a.bias ? a.bias[n + e] : 0.0f;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int64_t c = n + e < a.n ? n + e : a.n - 1;
        ws[j][e] = a.ws[c];
        b[j][e] = a.bias ? a.bias[c] : 0.0f;
      }
    }
  }
  constexpr int V = 16 / (int)sizeof(OT), COLS = BN / WN, PITCH = COLS * (int)sizeof(OT) + 16, PER_ROW = COLS / V;
  static_assert(WM * WN * 32 * PITCH <= 2 * STAGE, "the stages hold the epilogue");
  __syncthreads();
  uint8_t* own = lds + wave * (32 * PITCH);
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t mb = m0 + wm * (BM / WM) + i * 32, m = mb + lr;
    const float xs = a.xs ? a.xs[m < a.rows ? m : a.rows - 1] : 1.0f;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 16; e += V) {
        struct alignas(16) { OT v[V]; } y;
#pragma unroll
        for (int q = 0; q < V; ++q) {
          int v = acc[i][j][e + q];
          if constexpr (U8) v += lack[j][e + q];
          y.v[q] = linear_out<OT>(v, xs, ws[j][e + q], b[j][e + q], a.relu);
        }
        *(decltype(y)*)(own + lr * PITCH + (j * 32 + half * 16 + e) * (int)sizeof(OT)) = y;
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int c = lane; c < 32 * PER_ROW; c += 64) {
      const int row = c / PER_ROW, col = c % PER_ROW * V;
      struct alignas(16) { OT v[V]; } y = *(const decltype(y)*)(own + row * PITCH + col * (int)sizeof(OT));
      if (mb + row < a.rows) linear_put<OT, V>(a, mb + row, n0 + wn * COLS + col, y.v);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

}  // namespace ops
}  // namespace tg
