// tg_beam_select, tg_beam_reorder: one step of a beam search over beams and entries, and the rows that follow their beams.
#pragma once
#include "../../include/tetris_gym_hip.h"
#include "tg_op_common.h"

namespace tg {
namespace ops {

struct SelectArgs {
  const void* x;
  const float* scores;
  const uint8_t* mask;      // or null
  const uint8_t* finished;  // or null
  float* out_scores;
  int32_t* parents;
  int32_t* tokens;
  int64_t lg, lk, mg, mk;
  int64_t groups;
  int k, v, beams, pad, norm;
};

// e^d for d <= 700 (NaN: e^-700; the callers look for NaN themselves) to 1.1e-12 of its value, in 16 instructions: d log2(e) = n + f,
// |f| <= 1/2; 2^f is the Chebyshev interpolation of degree 8 on [-1/2, 1/2], and n is added to its exponent.  Below -700 it stays at
// 1e-304, which is nothing beside the largest term's 1.
__device__ __forceinline__ double exp64(double d) {
  const double big = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are the nearest integer
  const double t = fmax(d, -700.0) * 1.4426950408889634, z = t + big, f = t - (z - big);
  double p = 0x1.63d1279ae38e4p-20;
  p = fma(p, f, 0x1.00dc4a6dc0000p-16);
  p = fma(p, f, 0x1.4308ac93a7c72p-13);
  p = fma(p, f, 0x1.5d8745a6f2c72p-10);
  p = fma(p, f, 0x1.3b2ab7181339fp-7);
  p = fma(p, f, 0x1.c6b08dd6fd627p-5);
  p = fma(p, f, 0x1.ebfbdff823d48p-3);
  p = fma(p, f, 0x1.62e42fef84cedp-1);
  p = fma(p, f, 1.0);
  const uint64_t u = (uint64_t)__double_as_longlong(p);
  return __longlong_as_double((long long)(u + ((uint64_t)(uint32_t)(uint64_t)__double_as_longlong(z) << 52)));
}

// ln(s) for positive normal s = 2^e h, h in [0.7, 1.4): the hardware's float32 logarithm y of h, then one step of Newton's method to the
// third order in what it lacks (h e^-y = 1 + z, |z| < 2^-16: z - z^2/2 leaves z^3/3 < 2e-15); the error is that of exp64.  ln(1) is 0
// exactly: a beam with one allowed entry keeps its score.
__device__ __forceinline__ double log64(double s) {
  int e;
  double h = frexp(s, &e);
  if (h < 0.7) {
    h += h;
    --e;
  }
  const double y = (double)(__builtin_amdgcn_logf((float)h) * 0.693147180559945f);
  const double z = fma(h, exp64(-y), -1.0);
  return fma((double)e, 0x1.62e42fefa39efp-1, y + fma(-0.5 * z, z, z));
}

// A candidate as two words, larger = better, {0, .} = none: the score, then (beam, logit, entry) — within a beam the score never falls
// with the logit, so entries of one beam rank by their logit, and by their place where that is equal.
struct Key { uint64_t s, r; };
__device__ __forceinline__ bool better(const Key& a, const Key& b) { return a.s > b.s || (a.s == b.s && a.r > b.r); }
__device__ __forceinline__ uint64_t key_rest(int row, uint32_t xo, int v) {
  return ((uint64_t)(63 - row) << 56) | ((uint64_t)xo << 24) | (uint64_t)(0xFFFFFF - v);
}
__device__ __forceinline__ Key make_key(double c, int row, uint32_t xo, int v) {
  Key k;
  k.s = c > -__builtin_inf() ? order_f64(c) : 0;  // (NaN and -inf are no candidates)
  k.r = key_rest(row, xo, v);
  return k;
}
__device__ __forceinline__ void put_result(const SelectArgs& a, int64_t o, const Key& k) {
  const bool none = k.s == 0;
  a.out_scores[o] = none ? -__builtin_inff() : (float)unorder_f64(k.s);
  a.parents[o] = none ? -1 : 63 - (int)(k.r >> 56);
  a.tokens[o] = none ? -1 : 0xFFFFFF - (int)(k.r & 0xFFFFFF);
}
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, int l) {  // the value of lane l (uniform), in scalar registers
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, l) | ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), l) << 32);
}
__device__ __forceinline__ uint64_t max_u64(uint64_t a, uint64_t b) { return a > b ? a : b; }

__device__ __forceinline__ float lane_f32(float v, int l) { return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), l)); }

// A bound that at least `beams` (or all) of the wave's lane maxima reach: with up to 16 beams the beams-th largest of the 16 maxima of
// four lanes, else of the 64 lane maxima, by counting for each how many are larger.  m = -inf: the lane has nothing; none then passes
// a bound above -inf.
__device__ __forceinline__ float wave_bound(float m, int beams) {
  auto hi = [](float a, float b) { return a > b ? a : b; };
  const bool quads = beams <= 16;
  if (quads) m = group_reduce<4>(m, hi);
  int larger = 0;
  if (quads) {
#pragma unroll
    for (int l = 0; l < 64; l += 4) larger += lane_f32(m, l) > m;
  } else {
    for (int l = 0; l < 64; ++l) larger += lane_f32(m, l) > m;
  }
  // of the values with fewer than `beams` larger ones the smallest: equal values count once, so this is never above the beams-th
  return group_reduce<64>(larger < beams ? m : __builtin_inff(), [](float a, float b) { return a < b ? a : b; });
}

// A candidate before it is ranked: its score (-inf or NaN: none), its logit, and its beam and entry (row << 24 | entry).
struct Cand { double c; float x; uint32_t at; };
__device__ __forceinline__ Key key_of(const Cand& a) { return make_key(a.c, (int)(a.at >> 24), order_f32(a.x), (int)(a.at & 0xFFFFFF)); }

// Of N candidates per lane the best `beams` of the wave, handed to put(rank, key) in descending order; returns how many there are.
// The bound is taken over the scores rounded to float32 (rounding keeps their order, so nothing that belongs to the best is lost);
// what reaches it is packed into one candidate per lane through LDS (64 per wave) and ranked by counting; where more than 64 reach it
// (many equal ones, many beams), the best is taken out `beams` times instead.
template <int N, class F> __device__ __forceinline__ int wave_top(const Cand (&k)[N], int beams, Cand* lds, F put) {
  const int lane = threadIdx.x & 63;
  constexpr float low = -3.402823466e38f;  // (a score below the float range is still one)
  float c[N], m = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    c[i] = k[i].c > -__builtin_inf() ? fmaxf((float)k[i].c, low) : -__builtin_inff();
    m = fmaxf(m, c[i]);
  }
  const float bound = fmaxf(wave_bound(m, beams), low);
  int n = 0, at[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint64_t b = __ballot(c[i] >= bound);
    at[i] = n + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0));
    n += (int)__popcll(b);
  }
  if (n <= 64) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (c[i] >= bound) lds[at[i]] = k[i];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    Key key = {0, 0};
    float f = -__builtin_inff();
    if (lane < n) {
      const Cand o = lds[lane];
      key = key_of(o);
      f = (float)o.c;
    }
    int rank = 0, same = 0;
    for (int l = 0; l < n; ++l) {
      const float o = lane_f32(f, l);
      rank += o > f;
      same += o == f;
    }
    if (__ballot(lane < n && same > 1)) {  // equal in float32: by the whole key
      rank = 0;
      for (int l = 0; l < n; ++l) rank += better(Key{lane_u64(key.s, l), lane_u64(key.r, l)}, key);
    }
    if (lane < n && rank < beams) put(rank, key);
    __builtin_amdgcn_wave_barrier();
    return n < beams ? n : beams;
  }
  Key all[N];
#pragma unroll
  for (int i = 0; i < N; ++i) all[i] = key_of(k[i]);
  for (int b = 0; b < beams; ++b) {
    Key best = {0, 0};
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (better(all[i], best)) best = all[i];
    const uint64_t s = group_reduce<64>(best.s, max_u64), r = group_reduce<64>(best.s == s ? best.r : (uint64_t)0, max_u64);
    if (s == 0) return b;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (all[i].s == s && all[i].r == r) {
        put(b, all[i]);
        all[i].s = 0;
      }
  }
  return beams;
}

// Small searches: a wave per group, L = the power of two below 64 / K lanes per beam, N entries per lane (V <= L * N).  The log-sum of
// a beam is a reduction over its L lanes.  Everything stays in registers; the input is read once.  Bound by vector instructions: 8 192
// groups x 8 beams x 40 entries in f32 under a mask (13 MB) 11.8 us at 567 of them per wave, 8 us without log-probabilities; one group 2.6 us.
template <class T, int N> __global__ __launch_bounds__(256) void select_small_kernel(const SelectArgs a, int shift) {
  __shared__ Cand lds[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t g = (int64_t)blockIdx.x * 4 + wave;
  if (g >= a.groups) return;
  const int L = 1 << shift, j = lane >> shift, sub = lane & (L - 1);
  const bool here = j < a.k;
  const int jj = here ? j : 0;
  const T* x = (const T*)a.x + g * a.lg + jj * a.lk;
  T raw[N];
  uint32_t at[N], ok[N];  // (every load in front of the first use: a wave waits for memory once)
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int v = sub + i * L;
    at[i] = v < a.v ? v : 0;
    raw[i] = x[at[i]];
    ok[i] = 1;
  }
  const float sc = a.scores[g * a.k + jj];
  uint32_t fin = 0;
  if (a.finished) fin = a.finished[g * a.k + jj];
  if (a.mask) {
    const uint8_t* mask = a.mask + g * a.mg + jj * a.mk;
#pragma unroll
    for (int i = 0; i < N; ++i) ok[i] = mask[at[i]];
  }
  const bool done = fin != 0;
  float e[N];
#pragma unroll
  for (int i = 0; i < N; ++i) e[i] = here && !done && ok[i] != 0 && sub + i * L < a.v ? to_f32(raw[i]) : -__builtin_inff();
  double md = 0, ls = 0;  // the log-sum as maximum + logarithm: (x - md) - ls is the same for rows that differ by a constant
  if (a.norm) {
    float m = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, e[i]);
    auto fm = [](float p, float q) { return fmaxf(p, q); };
    if (L > 1) m = fm(m, xor_lane<1>(m));
    if (L > 2) m = fm(m, xor_lane<2>(m));
    if (L > 4) m = fm(m, xor_lane<4>(m));
    if (L > 8) m = fm(m, xor_lane<8>(m));
    if (L > 16) m = fm(m, xor_lane<16>(m));
    if (L > 32) m = fm(m, xor_lane<32>(m));
    double s = 0;
    md = m;
    bool nan = m == __builtin_inff();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      nan |= e[i] != e[i];
      s += exp64((double)e[i] - md);  // (m = -inf: the beam has no candidate, whatever this is)
    }
    if (nan) s = __builtin_nan("");  // (not a distribution: no candidate)
    if (L > 1) s += xor_lane<1>(s);
    if (L > 2) s += xor_lane<2>(s);
    if (L > 4) s += xor_lane<4>(s);
    if (L > 8) s += xor_lane<8>(s);
    if (L > 16) s += xor_lane<16>(s);
    if (L > 32) s += xor_lane<32>(s);
    ls = log64(s);
  }
  Cand k[N];
#pragma unroll
  for (int i = 0; i < N; ++i)
    k[i] = {e[i] > -__builtin_inff() ? (double)sc + (((double)e[i] - md) - ls) : -__builtin_inf(), e[i], ((uint32_t)jj << 24) + (uint32_t)(sub + i * L)};
  if (here && done && sub == 0) k[0] = {(double)sc, 0.0f, ((uint32_t)j << 24) + (uint32_t)a.pad};
  const int64_t o = g * a.beams;
  const int n = wave_top(k, a.beams, lds[wave], [&](int rank, const Key& c) { put_result(a, o + rank, c); });
  if (lane >= n && lane < a.beams) put_result(a, o + lane, Key{0, 0});
}

// Large searches, first step: a workgroup per (beam, chunk of 256 * E entries), the chunk in registers: its maximum, its sum of
// exponentials against that maximum, and its best `beams` entries by (logit, place).  32 x 8 x 32 768 in bf16 (17 MB): 14.5 us, 7 of them
// the issue of 943 vector instructions per wave (5 us without the exponentials, 3 without the list); chunks of 4 096: 15.0, 2 048: 18.0.
// What reaches a wave's bound is ranked by counting, so the list is kept short: where many equal logits (a clipped or a constant row), rising
// ones or many beams bring more than kSelectList entries, every wave first narrows its bound until at most kSelectWave remain.
// 32 x 8 x 32 768 in bf16, whole calls at 8, 16, 64 beams: random logits 20, 37, 114 us, all equal 44, 53, 363 (ranking the
// whole chunk instead: 7 930 and 8 250 at 16 and 64).
constexpr int kSelectList = 256, kSelectWave = kSelectList / 4;
static_assert(kSelectWave >= TG_OPS_MAX_BEAMS, "a wave lists its best `beams` at least");
struct SelectPart { double s; float m; int n; };  // then uint64_t[beams]: order(logit) << 32 | ~entry, descending, n of them
__device__ __host__ __forceinline__ int64_t select_part_bytes(int beams) { return 16 + 8 * (int64_t)beams; }

template <class T, int E> __global__ __launch_bounds__(256) void select_chunk_kernel(const SelectArgs a, int chunks, uint8_t* ws) {
  constexpr int V = 16 / (int)sizeof(T), NV = E / V;
  __shared__ uint64_t list[kSelectList];
  __shared__ float wm[4];
  __shared__ double wsum[4];
  __shared__ int count;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int64_t row = blockIdx.x / chunks, g = row / a.k;
  const int chunk = blockIdx.x % chunks, j = (int)(row % a.k);
  uint8_t* part = ws + (int64_t)blockIdx.x * select_part_bytes(a.beams);
  SelectPart* head = (SelectPart*)part;
  uint64_t* keys = (uint64_t*)(part + 16);
  const float score = a.scores[row];
  const uint8_t done = a.finished ? a.finished[row] : 0;
  if (t == 0) count = 0;
  const T* x = (const T*)a.x + g * a.lg + j * a.lk;
  const uint8_t* mask = a.mask + g * a.mg + j * a.mk;  // (only where a.mask is)
  const int v0 = chunk * (256 * E) + t * V;
  float e[E];
  if ((chunk + 1) * (256 * E) <= a.v) {  // a whole chunk: every load in front of the first use
    v4i u[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) u[i] = load16(x + v0 + i * 256 * V);
    struct __attribute__((packed, aligned(1))) Bytes { uint8_t b[V]; } ok[NV];
    if (a.mask) {
#pragma unroll
      for (int i = 0; i < NV; ++i) ok[i] = *(const Bytes*)(mask + v0 + i * 256 * V);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      T h[V];
      __builtin_memcpy(h, &u[i], 16);
#pragma unroll
      for (int q = 0; q < V; ++q) e[i * V + q] = to_f32(h[q]);
    }
    if (a.mask) {
#pragma unroll
      for (int i = 0; i < E; ++i) e[i] = ok[i / V].b[i % V] ? e[i] : -__builtin_inff();
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int v = v0 + (i / V) * 256 * V + i % V;
      e[i] = v < a.v && (!a.mask || mask[v]) ? to_f32(x[v]) : -__builtin_inff();
    }
  }
  if (done || !(score > -__builtin_inff())) {  // (offers nothing of its own; asked behind the loads, not in front of them)
    if (t == 0) *head = {0.0, -__builtin_inff(), 0};
    return;
  }
  // The sum starts as soon as the lane's first entries are there: against their maximum `ref`, not the chunk's (float64 holds e^600 of
  // it; an entry further above moves the reference), and the lanes' sums are brought to the chunk's maximum at the end.
  float lm = -__builtin_inff(), ref = 0;
  double s = 0;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float vm = -__builtin_inff();
#pragma unroll
    for (int q = 0; q < V; ++q) vm = fmaxf(vm, e[i * V + q]);  // (a NaN is not in it)
    if (a.norm) {
      if (lm == -__builtin_inff()) ref = vm > -__builtin_inff() ? vm : 0.0f;
      const bool far = vm - ref > 600.0f;  // (also where vm is infinite)
      if (__ballot(far)) {
        if (far) {
          s *= exp64((double)ref - (double)vm);
          ref = vm;
        }
      }
      const double rd = ref;
#pragma unroll
      for (int q = 0; q < V; ++q) {
        nan |= e[i * V + q] != e[i * V + q];
        s += exp64((double)e[i * V + q] - rd);
      }
    }
    lm = fmaxf(lm, vm);
  }
  float m = group_reduce<64>(lm, [](float p, float q) { return fmaxf(p, q); });
  if (lane == 0) wm[wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3]));
  if (a.norm) {
    s = lm > -__builtin_inff() ? s * exp64((double)ref - (double)m) : 0.0;  // (a lane without entries summed e^-700 each)
    if (nan || m == __builtin_inff()) s = __builtin_nan("");
    s = group_reduce<64>(s, [](double p, double q) { return p + q; });
    if (lane == 0) wsum[wave] = s;
  }
  // what reaches the wave's bound is listed, as (logit, place)
  auto entry = [&](int i) { return v0 + (i / V) * 256 * V + i % V; };
  auto key = [&](float f, int v) { return ((uint64_t)order_f32(f) << 32) | (uint32_t)~v; };
  const float bf = fmaxf(wave_bound(lm, a.beams), -3.402823466e38f);
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const bool in = e[i] >= bf;
    if (__ballot(in)) {
      if (in) {
        const int at = atomicAdd(&count, 1);
        if (at < kSelectList) list[at] = key(e[i], entry(i));
      }
    }
  }
  __syncthreads();
  if (count > kSelectList) {
    __syncthreads();
    if (t == 0) count = 0;
    __syncthreads();
    // The bound rises, by halving what lies between it and the wave's largest, as long as `beams` entries reach it; where it ends among
    // equal logits with too many of them, those behind a place that is found likewise stay out.
    auto reach = [&](auto in) {
      int n = 0;
#pragma unroll
      for (int i = 0; i < E; ++i) n += (int)__popcll(__ballot(in(i)));
      return n;
    };
    float f = bf;
    int last = 256 * E, n = reach([&](int i) { return e[i] >= f; });
    uint32_t lo = order_f32(bf), hi = order_f32(group_reduce<64>(lm, [](float p, float q) { return fmaxf(p, q); }));
    while (n > kSelectWave && lo < hi) {
      const uint32_t mid = lo + (hi - lo + 1) / 2;
      const float g = unorder_f32(mid);
      const int more = reach([&](int i) { return e[i] >= g; });
      if (more >= a.beams) {
        lo = mid;
        f = g;
        n = more;
      } else {
        hi = mid - 1;
      }
    }
    if (n > kSelectWave) {  // (fewer than `beams` are above f: it cannot rise)
      const int want = a.beams - reach([&](int i) { return e[i] > f; });
      int from = chunk * (256 * E), to = from + 256 * E - 1;  // the place of the want-th of those at f
      while (from < to) {
        const int mid = from + (to - from) / 2;
        const int in_lane = mid - v0;  // (against a constant for each entry)
        if (reach([&](int i) { return e[i] == f && (i / V) * 256 * V + i % V <= in_lane; }) >= want) to = mid;
        else from = mid + 1;
      }
      last = to - v0;
    }
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (e[i] > f || (e[i] == f && (i / V) * 256 * V + i % V <= last)) list[atomicAdd(&count, 1)] = key(e[i], entry(i));
  }
  __syncthreads();
  const int n = count, keep = n < a.beams ? n : a.beams;
  for (int i = t; i < n; i += 256) {
    const uint64_t k = list[i];
    int rank = 0;
    for (int l = 0; l < n; ++l) rank += list[l] > k;
    if (rank < keep) keys[rank] = k;
  }
  if (t == 0) *head = {a.norm ? wsum[0] + wsum[1] + wsum[2] + wsum[3] : 0.0, m, keep};
}

// ... second step: a workgroup per group puts the chunks' sums together, a wave per beam and a lane per chunk; its first wave then goes
// through the candidates in rounds of 256, the first entries of all lists before the second ones, so that later rounds soon hold
// nothing better than the `beams` already found.  Bound by latency (one small workgroup per group): the first round's candidates are
// asked for at the start.
__global__ __launch_bounds__(1024) void select_merge_kernel(const SelectArgs a, int chunks, const uint8_t* ws) {
  constexpr int N = 4;
  __shared__ Cand lds[64];
  __shared__ Key top[64];
  __shared__ double row_max[64], row_log[64];
  __shared__ float score[64];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, waves = blockDim.x >> 6;
  const int64_t g = blockIdx.x, pb = select_part_bytes(a.beams);
  const uint8_t* base = ws + g * a.k * chunks * pb;
  const uint32_t lists = (uint32_t)(a.k * chunks), total = lists * (uint32_t)a.beams;
  auto part = [&](uint32_t l) { return (const SelectPart*)(base + (int64_t)l * pb); };
  uint64_t u[N];
  uint32_t row[N];
  auto fetch = [&](uint32_t c0) {  // candidates of all lists, 0 where a list is shorter
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t c = c0 + 64 * i + lane;
      u[i] = row[i] = 0;
      if (c < total) {
        const uint32_t rank = c / lists, l = c - rank * lists;
        row[i] = l / (uint32_t)chunks;
        u[i] = ((const uint64_t*)(part(l) + 1))[rank];
        if ((int)rank >= part(l)->n) u[i] = 0;
      }
    }
  };
  bool done = false;
  if (wave == 0) {
    fetch(0);
    if (lane < a.k) {
      score[lane] = a.scores[g * a.k + lane];
      done = a.finished && a.finished[g * a.k + lane];
      if (!a.norm) row_max[lane] = row_log[lane] = 0;
    }
  }
  if (a.norm) {
    for (int j = wave; j < a.k; j += waves) {
      float m = -__builtin_inff();
      double s = 0;
      for (int c = lane; c < chunks; c += 64) {
        const SelectPart h = *part((uint32_t)(j * chunks + c));
        if (h.m > m) {
          s *= exp64((double)m - (double)h.m);  // (m = -inf: s is 0)
          m = h.m;
        }
        if (h.s != 0.0) s += h.s * exp64((double)h.m - (double)m);
      }
      const float all = group_reduce<64>(m, [](float p, float q) { return fmaxf(p, q); });
      if (s != 0.0) s *= exp64((double)m - (double)all);
      s = group_reduce<64>(s, [](double p, double q) { return p + q; });
      if (lane == 0) {
        row_max[j] = all;
        row_log[j] = log64(s);
      }
    }
  }
  __syncthreads();
  if (wave) return;
  int found = 0;
  Key bottom = {0, 0};  // the worst of the `beams` found so far, or none
  for (uint32_t i0 = 0;; i0 += 64 * N) {
    Cand k[N + 1];
    bool any = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float x = unorder_f32((uint32_t)(u[i] >> 32));
      k[i] = {u[i] ? (double)score[row[i]] + (((double)x - row_max[row[i]]) - row_log[row[i]]) : -__builtin_inf(), x, (row[i] << 24) | ~(uint32_t)u[i]};
      if (found == a.beams && !better(key_of(k[i]), bottom)) k[i].c = -__builtin_inf();
      any |= k[i].c > -__builtin_inf();
    }
    // behind them a finished beam's one candidate, or what was found before
    k[N] = {-__builtin_inf(), 0.0f, 0};
    if (i0 == 0) {
      if (done) k[N] = {(double)score[lane], 0.0f, ((uint32_t)lane << 24) | (uint32_t)a.pad};
      any |= done;
    } else if (lane < found) {
      const Key c = top[lane];
      k[N] = {unorder_f64(c.s), unorder_f32((uint32_t)(c.r >> 24)), ((uint32_t)(63 - (int)(c.r >> 56)) << 24) | (uint32_t)(0xFFFFFF - (c.r & 0xFFFFFF))};
    }
    const bool more = i0 + 64 * N < total;
    if (more) fetch(i0 + 64 * N);
    if (__ballot(any)) {
      __builtin_amdgcn_wave_barrier();
      found = wave_top(k, a.beams, lds, [&](int rank, const Key& c) { top[rank] = c; });
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (found == a.beams) bottom = top[a.beams - 1];
    }
    if (!more) break;
  }
  if (lane < a.beams) put_result(a, g * a.beams + lane, lane < found ? top[lane] : Key{0, 0});
}

// which of them, by sizes alone (the workspace goes by it)
struct SelectPlan { bool small; int shift, per_lane, e, chunks; };
inline SelectPlan select_plan(int64_t groups, int64_t k, int64_t v) {
  SelectPlan p{};
  p.shift = 6;
  while (k << p.shift > 64) --p.shift;
  const int64_t per = (v + (1 << p.shift) - 1) >> p.shift;
  if (per <= 16) {
    p.small = true;
    p.per_lane = (int)per;
    return p;
  }
  p.e = v <= 2048 ? 8 : v <= 4096 ? 16 : 32;
  while (p.e > 8 && groups * k * ((v + 256 * p.e - 1) / (256 * p.e)) < 1024) p.e /= 2;  // enough workgroups for four per compute unit
  p.chunks = (int)((v + 256 * p.e - 1) / (256 * p.e));
  return p;
}

// ---- reorder -------------------------------------------------------------------------------------------------------------------
// An item is gp groups x kout beams x cb columns (units of 1 << shift bytes) of one array, at most 64 * kReorderReg units: a wave takes
// the whole item into registers before it stores any of it, and columns of a row do not depend on each other, so the rows of a
// group may be permuted in place.  Rows go in units of 16 bytes at whatever address they start, and what is left of them (below 16
// bytes) as an array of its own.  Bound by memory: 65 536 envs of 320 bytes in four arrays (42 MB) 10.5 us = 4.0 TB/s (in
// units of 8 bytes 11.4), 32 rows of 1 MiB (67 MB) 13.0 us = 5.2 TB/s; in place, whole calls, 9.8 and 10.7.
constexpr int kReorderReg = 8, kReorderMax = 48;
struct ReorderArray {
  const uint8_t* src;
  uint8_t* dst;
  int64_t src_stride, dst_stride;  // bytes
  int64_t units;                   // of a row
  int64_t last;                    // where the last of them starts: it may overlap the one before (an item then holds whole rows)
  uint32_t blocks;                 // column blocks
  int cb, gp, shift;
  uint32_t mul_cb, mul_out;        // t / cb = t * mul_cb >> 21, likewise / beams out (t < 512)
};
struct ReorderArgs {
  ReorderArray a[kReorderMax];
  uint32_t first[kReorderMax];  // first item; 2^32 - 1 behind the last array
  const int32_t* parents;
  int64_t groups;
  uint32_t items;
  uint32_t base;  // the launch's first item
  int n, kin, kout, in_place;
};
static_assert(sizeof(ReorderArgs) <= 4096, "kernel arguments");

template <class U> struct __attribute__((packed, aligned(1))) AnyPlace { U v; };

template <class U> __device__ __forceinline__ void reorder_item(const ReorderArray& a, const ReorderArgs& p, uint32_t item, int lane) {
  const int64_t g0 = (int64_t)(item / a.blocks) * a.gp, c0 = (int64_t)(item % a.blocks) * a.cb;
  int parent[kReorderReg];
  int64_t to[kReorderReg];
  U v[kReorderReg];
#pragma unroll
  for (int i = 0; i < kReorderReg; ++i) {
    const uint32_t t = (uint32_t)(i * 64 + lane);
    const uint32_t rg = (t * a.mul_cb) >> 21, c = t - rg * a.cb;        // row of the item, column
    const uint32_t dg = (rg * a.mul_out) >> 21, r = rg - dg * p.kout;   // group of the item, beam
    const int64_t row = g0 * p.kout + rg;
    parent[i] = -1;
    to[i] = 0;
    if ((int)dg < a.gp && g0 + dg < p.groups && c0 + c < a.units) {
      const int q = p.parents[row];
      const int64_t at = (c0 + c) << a.shift;
      to[i] = row * a.dst_stride + (at < a.last ? at : a.last);
      parent[i] = p.in_place && q == (int)r ? -1 : q;
    }
  }
#pragma unroll
  for (int i = 0; i < kReorderReg; ++i) {
    const uint32_t t = (uint32_t)(i * 64 + lane);
    const uint32_t rg = (t * a.mul_cb) >> 21, c = t - rg * a.cb, dg = (rg * a.mul_out) >> 21;
    if ((uint32_t)parent[i] < (uint32_t)p.kin) {  // (negative ones are large)
      const int64_t at = (c0 + c) << a.shift;
      v[i] = ((const AnyPlace<U>*)(a.src + ((g0 + dg) * p.kin + parent[i]) * a.src_stride + (at < a.last ? at : a.last)))->v;
    }
  }
  if (p.in_place) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // every load of the wave is back before its first store
#pragma unroll
  for (int i = 0; i < kReorderReg; ++i)
    if ((uint32_t)parent[i] < (uint32_t)p.kin) ((AnyPlace<U>*)(a.dst + to[i]))->v = v[i];
}

__global__ __launch_bounds__(256) void reorder_kernel(const ReorderArgs p) {
  const uint32_t item = p.base + blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (item >= p.items) return;
  int k = -1;
#pragma unroll
  for (int i = 0; i < kReorderMax; ++i) k += item >= p.first[i];
  const ReorderArray& a = p.a[k];
  const int lane = threadIdx.x & 63;
  const uint32_t it = item - p.first[k];
  switch (a.shift) {
    case 4: reorder_item<v4i>(a, p, it, lane); break;
    case 3: reorder_item<uint64_t>(a, p, it, lane); break;
    case 2: reorder_item<uint32_t>(a, p, it, lane); break;
    case 1: reorder_item<uint16_t>(a, p, it, lane); break;
    default: reorder_item<uint8_t>(a, p, it, lane); break;
  }
}

// ---- bookkeeping of a search around a transition: a thread per environment, bound by the launch --------------------------------------
__global__ __launch_bounds__(256) void advance_kernel(const int32_t* parents, const int32_t* tokens, const float* gain_in, float* gain_out,
                                                      int32_t* actions, int64_t n, int beams) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int p = parents[i];
  const bool ok = p >= 0 && p < beams;
  gain_out[i] = ok ? gain_in[i / beams * beams + p] : -__builtin_inff();
  actions[i] = ok ? tokens[i] : 0;
}
__global__ __launch_bounds__(256) void collect_kernel(const tg_step_out* out, float* gain, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  gain[i] = out[i].terminated ? -__builtin_inff() : gain[i] + out[i].reward;
}

}  // namespace ops
}  // namespace tg
