// tg_beam_select, tg_beam_reorder: one step of a beam search over beams and entries, and the rows that follow their beams.
#pragma once
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

// a candidate in the order of the result: better() is a strict total order (within a beam the score never falls with the logit)
struct Cand { double s; float x; int row, v; };
__device__ __forceinline__ bool better(const Cand& a, const Cand& b) {
  if (a.row == b.row) return a.x > b.x || (a.x == b.x && a.v < b.v);
  return a.s > b.s || (a.s == b.s && a.row < b.row);
}
__device__ __forceinline__ Cand cand_none() { return {-__builtin_inf(), -__builtin_inff(), 1 << 30, 1 << 30}; }

// One workgroup per group: the rows' log-sums, then one scan per result for the best candidate behind the last one.
template <class T> __global__ __launch_bounds__(256) void select_scan_kernel(const SelectArgs a) {
  __shared__ double lse[64], red[4];
  __shared__ float redf[4];
  __shared__ Cand best[4];
  const int64_t g = blockIdx.x;
  const int t = threadIdx.x, wave = t >> 6;
  const T* x = (const T*)a.x + g * a.lg;
  const uint8_t* mask = a.mask ? a.mask + g * a.mg : nullptr;
  auto at = [&](int j, int i) {  // the logit of an allowed entry; what is not allowed reads as -inf
    if (mask && !mask[j * a.mk + i]) return -__builtin_inff();
    return to_f32(x[j * a.lk + i]);
  };
  for (int j = 0; j < a.k; ++j) {
    double L = 0;
    if (a.norm) {
      float m = -__builtin_inff();
      bool nan = false;
      for (int i = t; i < a.v; i += 256) {
        const float e = at(j, i);
        nan |= e != e;
        m = fmaxf(m, e);
      }
      m = group_reduce<64>(m, [](float p, float q) { return fmaxf(p, q); });
      if ((t & 63) == 0) redf[wave] = m;
      __syncthreads();
      m = fmaxf(fmaxf(redf[0], redf[1]), fmaxf(redf[2], redf[3]));
      double s = nan ? __builtin_nan("") : 0.0;
      if (m > -__builtin_inff())
        for (int i = t; i < a.v; i += 256) s += exp((double)at(j, i) - (double)m);  // (m = +inf: NaN)
      s = group_reduce<64>(s, [](double p, double q) { return p + q; });
      if ((t & 63) == 0) red[wave] = s;
      __syncthreads();
      s = red[0] + red[1] + red[2] + red[3];
      L = (double)m + log(s);
      __syncthreads();
    }
    if (t == 0) lse[j] = L;
  }
  __syncthreads();
  Cand last = {__builtin_inf(), __builtin_inff(), -1, -1};
  for (int b = 0; b < a.beams; ++b) {
    Cand mine = cand_none();
    for (int j = 0; j < a.k; ++j) {
      const float sc = a.scores[g * a.k + j];
      if (a.finished && a.finished[g * a.k + j]) {
        const Cand c = {(double)sc, 0.0f, j, a.pad};
        if (t == 0 && c.s > -__builtin_inf() && better(last, c) && better(c, mine)) mine = c;
        continue;
      }
      for (int i = t; i < a.v; i += 256) {
        const float e = at(j, i);
        const Cand c = {(double)sc + ((double)e - lse[j]), e, j, i};
        if (c.s > -__builtin_inf() && e > -__builtin_inff() && better(last, c) && better(c, mine)) mine = c;
      }
    }
    auto pick = [](Cand p, const Cand& q) { return better(q, p) ? q : p; };
    for (int d = 32; d; d >>= 1) {
      Cand o;
      o.s = __shfl_xor(mine.s, d);
      o.x = __shfl_xor(mine.x, d);
      o.row = __shfl_xor(mine.row, d);
      o.v = __shfl_xor(mine.v, d);
      mine = pick(mine, o);
    }
    if ((t & 63) == 0) best[wave] = mine;
    __syncthreads();
    mine = pick(pick(pick(best[0], best[1]), best[2]), best[3]);
    __syncthreads();
    last = mine;
    const bool none = mine.row == 1 << 30;
    if (t == 0) {
      const int64_t o = g * a.beams + b;
      a.out_scores[o] = none ? -__builtin_inff() : (float)mine.s;
      a.parents[o] = none ? -1 : mine.row;
      a.tokens[o] = none ? -1 : mine.v;
    }
    if (none) last = cand_none();  // (nothing is behind it)
  }
}

// ---- reorder -------------------------------------------------------------------------------------------------------------------
// An item is gp groups x kin beams x cb columns (units of 1 << shift bytes) of one array, at most 64 * kReg units: a wave takes the
// whole item into registers before it stores any of it, and columns of a row do not depend on each other, so the rows of a group
// may be permuted in place.
constexpr int kReorderReg = 4, kReorderMax = 24;
struct ReorderArray {
  const uint8_t* src;
  uint8_t* dst;
  int64_t src_stride, dst_stride;  // bytes
  int64_t units;                   // of a row
  uint32_t first;                  // first item
  uint32_t blocks;                 // column blocks
  int cb, gp, shift;
  uint32_t mul_cb, mul_out;        // t / cb = t * mul_cb >> 20, likewise / beams out (t < 256)
};
struct ReorderArgs {
  ReorderArray a[kReorderMax];
  const int32_t* parents;
  int64_t groups;
  uint32_t items;
  int n, kin, kout, in_place;
};

template <class U> __device__ __forceinline__ void reorder_item(const ReorderArray& a, const ReorderArgs& p, uint32_t item, int lane) {
  const int64_t g0 = (int64_t)(item / a.blocks) * a.gp, c0 = (int64_t)(item % a.blocks) * a.cb;
  U v[kReorderReg];
  U* to[kReorderReg];
#pragma unroll
  for (int i = 0; i < kReorderReg; ++i) {
    const uint32_t t = (uint32_t)(i * 64 + lane);
    const uint32_t rg = (t * a.mul_cb) >> 20, c = t - rg * a.cb;        // row of the item, column
    const uint32_t dg = (rg * a.mul_out) >> 20, r = rg - dg * p.kout;   // group of the item, beam
    const int64_t g = g0 + dg, col = c0 + c;
    to[i] = nullptr;
    if ((int)dg < a.gp && g < p.groups && col < a.units) {
      const int from = p.parents[g * p.kout + r];
      if (from >= 0 && from < p.kin && !(p.in_place && from == (int)r)) {
        v[i] = *(const U*)(a.src + (g * p.kin + from) * a.src_stride + (col << a.shift));
        to[i] = (U*)(a.dst + (g * p.kout + r) * a.dst_stride + (col << a.shift));
      }
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // every load of the wave is back before its first store
#pragma unroll
  for (int i = 0; i < kReorderReg; ++i)
    if (to[i]) *to[i] = v[i];
}

__global__ __launch_bounds__(256) void reorder_kernel(const ReorderArgs p) {
  const uint32_t item = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (item >= p.items) return;
  int k = 0;
  while (k + 1 < p.n && item >= p.a[k + 1].first) ++k;
  const ReorderArray& a = p.a[k];
  const int lane = threadIdx.x & 63;
  switch (a.shift) {
    case 4: reorder_item<v4i>(a, p, item - a.first, lane); break;
    case 3: reorder_item<uint64_t>(a, p, item - a.first, lane); break;
    case 2: reorder_item<uint32_t>(a, p, item - a.first, lane); break;
    case 1: reorder_item<uint16_t>(a, p, item - a.first, lane); break;
    default: reorder_item<uint8_t>(a, p, item - a.first, lane); break;
  }
}

}  // namespace ops
}  // namespace tg
