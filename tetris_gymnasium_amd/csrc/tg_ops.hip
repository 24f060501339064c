// Host side of the operators' C ABI (include/tetris_gym_ops.h): checks, choice of a kernel, launch.
#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <tuple>

#include "../../include/tetris_gym_hip.h"
#include "../../include/tetris_gym_ops.h"
#include "tg_op_beam.h"
#include "tg_op_linear.h"
#include "tg_op_quantize.h"

using namespace tg::ops;

namespace {

thread_local char g_err[512];

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

// the call's device for the duration of the call
struct DeviceScope {
  int before = -1;
  hipError_t err;
  explicit DeviceScope(int device) {
    err = hipGetDevice(&before);
    if (err == hipSuccess && before != device) err = hipSetDevice(device);
    else before = -1;
  }
  ~DeviceScope() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};
#define ON_DEVICE(name, device)                                                                             \
  DeviceScope scope(device);                                                                                \
  if (scope.err != hipSuccess) {                                                                            \
    (void)hipGetLastError();                                                                                \
    return fail(TG_EHIP, name ": device %d: %s (there is no CPU fallback)", device, hipGetErrorString(scope.err)); \
  }

// A launch with its own answer: hipGetLastError would also report what another library left behind on this thread.
template <class... P, class... A> hipError_t launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t lds, hipStream_t stream, const A&... args) {
  std::tuple<P...> held{static_cast<P>(args)...};
  return std::apply([&](P&... p) {
    void* at[] = {(void*)&p...};
    return hipLaunchKernel((const void*)kernel, grid, block, at, lds, stream);
  }, held);
}
int launched(const char* name, hipError_t e) {
  if (e == hipSuccess) return TG_OK;
  (void)hipGetLastError();
  return fail(TG_EHIP, "%s: launch failed: %s", name, hipGetErrorString(e));
}

int type_size(int t) { return t <= kI8 ? 1 : t == kF32 ? 4 : 2; }
bool is_float(int t) { return t == kF32 || t == kF16 || t == kBF16; }

// Bytes from the first to behind the last element of [rows][cols] with a row stride, or of [groups][rows][cols] with a group stride too
// (sizes > 0, strides >= 0); -1 where they pass the 2^47 bytes that addresses reach: no memory holds such an array, and sums with it
// would leave 64 bits.
constexpr int64_t kAddresses = (int64_t)1 << 47;
int64_t span(int64_t rows, int64_t cols, int64_t stride, int64_t size, int64_t groups = 1, int64_t group_stride = 0) {
  const __int128 n = ((__int128)(groups - 1) * group_stride + (__int128)(rows - 1) * stride + cols) * size;
  return n > kAddresses ? -1 : (int64_t)n;
}
bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {
  return a && b && (const char*)a < (const char*)b + nb && (const char*)b < (const char*)a + na;
}
constexpr int64_t kMost = (int64_t)1 << 40;  // sizes and strides beyond a card's memory (what products of them reach: span)
constexpr int64_t kMaxGroups = 0x7FFFFFFF;
// A launch holds fewer than 2^32 threads along x, whatever the blocks are (with more, hipLaunchKernel has returned success here and run a
// part of the blocks): calls that need more are spread over several launches.
constexpr int64_t max_blocks(int threads) { return (int64_t)0xFFFFFFFF / threads; }

template <class F> hipError_t by_float(int t, F f) {
  if (t == kF32) return f(float{});
  if (t == kF16) return f(_Float16{});
  return f(bf16_t{});
}

constexpr int kUnits = 256;  // compute units

template <class OT, bool U8, int KS> hipError_t linear_rows(const LinearArgs& a, hipStream_t st) {
  const int64_t cols = (a.n + 63) / 64;
  const int shift = cols >= 4 ? 2 : cols == 2 ? 1 : 0, below = 4 >> shift;
  const int64_t gy = (cols + (1 << shift) - 1) >> shift, tiles = (a.rows + 15) / 16;
  // as many workgroups as stay resident (by the variant's registers), each with a run of tiles
  int64_t gx = (kUnits * (KS == 1 ? 3 : 2) + gy - 1) / gy;
  if (gx > (tiles + below - 1) / below) gx = (tiles + below - 1) / below;
  const int64_t inside = a.x_stride ? ((a.rows - 1) * a.x_stride + a.k - 64 * KS) / (16 * a.x_stride) : 0;
  return launch(linear_rows_kernel<OT, U8, KS>, dim3((unsigned)gx, (unsigned)gy), dim3(256), 0, st, a, shift, inside);
}

template <class OT, bool U8, int T, int U> hipError_t linear_few(const LinearArgs& a, hipStream_t st) {
  int waves = (int)((a.k + 255) / 256);
  waves = waves < 1 ? 1 : waves > 8 ? 8 : waves;
  const int kw = (int)((a.k + waves * 64 - 1) / (waves * 64)) * 64;
  return launch(linear_few_kernel<OT, U8, T, U>, dim3((unsigned)((a.n + 16 * T - 1) / (16 * T)), (unsigned)((a.rows + 16 * U - 1) / (16 * U))), dim3(64 * waves), 0, st, a, kw);
}

template <class OT, bool U8, int BM, int BN, int WM, int WN, bool AL> hipError_t linear_tile(const LinearArgs& a, hipStream_t st) {
  const int64_t mt = (a.rows + BM - 1) / BM, nt = (a.n + BN - 1) / BN;
  const int64_t most = max_blocks(WM * WN * 64) / nt;  // row tiles of one launch (nt <= 2^16)
  for (int64_t i = 0; i < mt; i += most) {
    LinearArgs b = a;
    b.x = a.x + i * BM * a.x_stride;
    b.xs = a.xs ? a.xs + i * BM : nullptr;
    b.out = (OT*)a.out + i * BM * a.out_stride;
    b.rows = a.rows - i * BM < most * BM ? a.rows - i * BM : most * BM;
    const int m = (int)((b.rows + BM - 1) / BM);
    const hipError_t e = launch(linear_tile_kernel<OT, U8, BM, BN, WM, WN, AL>, dim3((unsigned)(m * nt)), dim3(WM * WN * 64), 2 * (BM + BN) * 128, st, b, m, (int)nt);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// Times in us, back to back, bf16 out; rows x k x n.
template <class OT, bool U8> hipError_t linear_launch(const LinearArgs& a, hipStream_t st) {
  const auto tiles = [&](int64_t bm, int64_t bn) { return ((a.rows + bm - 1) / bm) * ((a.n + bn - 1) / bn); };
  // Few rows: the waves of a workgroup share K.  The widest variant that still gives every compute unit a workgroup: 64 x 4 096 x 8 192:
  // 15.3 (2, 4) against 17.7 (2, 2) and 30.7 (1, 1), but 64 x 1 024 x 1 024: 6.7, 4.8, 3.4.  Above 64 rows only where tiles would leave
  // most of the units idle: 128 x 1 024 x 1 024: 4.2 against 6.2; 128 x 4 096 x 8 192: 25.5 against 19.8.
  if (a.rows <= 64 || (a.rows <= 256 && tiles(64, 64) <= 64)) {
    if (a.rows > 32 && tiles(64, 32) >= kUnits) return linear_few<OT, U8, 2, 4>(a, st);
    if (a.rows > 16 && tiles(32, 32) >= kUnits) return linear_few<OT, U8, 2, 2>(a, st);
    if (tiles(16, 32) >= kUnits) return linear_few<OT, U8, 2, 1>(a, st);
    return linear_few<OT, U8, 1, 1>(a, st);
  }
  // Short rows: weights in registers: 65 536 x 200 x 256: 16.1 against 20.9 (tiles), x 256 x 256: 17.1 against 18.1; only where they would
  // multiply mostly columns that are not there, and 16-byte addresses allow it, tiles are better: x 256 x 40: 8.3 against 7.6.
  const bool al = (((uintptr_t)a.x | (uintptr_t)a.w | (uintptr_t)a.x_stride | (uintptr_t)a.w_stride | (uintptr_t)a.k) & 15) == 0;
  if (a.k <= 64) return linear_rows<OT, U8, 1>(a, st);
  if (a.k <= 128) return linear_rows<OT, U8, 2>(a, st);
  if (a.k <= 256 && !(al && a.n <= 64)) return linear_rows<OT, U8, 4>(a, st);
  // Tiles.  4 096 x 4 096 x 4 096 (256 of 256 x 256): 66 against 79 (128 x 128); 2 048 x 4 096 x 4 096 (128; 512 of 128 x 128): 52, 42, 53
  // (128 x 64); 1 024 x 4 096 x 4 096 (512 of 128 x 64): 29 (128 x 128), 27, 30 (64 x 64); 256 x 4 096 x 4 096: 19 (128 x 64), 15 (64 x 64).
  if (!al) return linear_tile<OT, U8, 128, 128, 2, 2, false>(a, st);
  if (a.n > 128 && a.k >= 512 && tiles(256, 256) >= kUnits) return linear_tile<OT, U8, 256, 256, 2, 4, true>(a, st);
  if (a.n > 64 && tiles(128, 128) >= 2 * kUnits) return linear_tile<OT, U8, 128, 128, 2, 2, true>(a, st);
  if (tiles(128, 64) >= 2 * kUnits) return linear_tile<OT, U8, 128, 64, 2, 2, true>(a, st);
  return linear_tile<OT, U8, 64, 64, 2, 2, true>(a, st);
}

}  // namespace

namespace tg { namespace ops { __attribute__((visibility("hidden"))) void set_error(const char* msg) { snprintf(g_err, sizeof(g_err), "%s", msg); } } }

extern "C" {

const char* tg_ops_last_error(void) { return g_err; }

int tg_linear_i8(int device, void* stream, const void* x, int x_type, int64_t rows, int64_t k, int64_t x_stride, const int8_t* w, int64_t n,
                 int64_t w_stride, const float* w_scale, const float* x_scale, const float* bias, int relu, void* out, int out_type,
                 int64_t out_stride) {
  if (x_type != kU8 && x_type != kI8) return fail(TG_EINVAL, "tg_linear_i8: x must be u8 or i8, got type %d", x_type);
  if (!is_float(out_type)) return fail(TG_EINVAL, "tg_linear_i8: out must be f32, f16 or bf16, got type %d", out_type);
  if (rows < 0 || n < 0 || k < 0 || rows > kMost || n > kMost) return fail(TG_EINVAL, "tg_linear_i8: bad sizes (rows %lld, k %lld, n %lld)", (long long)rows, (long long)k, (long long)n);
  if (k > TG_OPS_MAX_K) return fail(TG_EINVAL, "tg_linear_i8: k = %lld, the 32-bit sum is exact up to %d", (long long)k, TG_OPS_MAX_K);
  if (rows == 0 || n == 0) return TG_OK;
  if ((rows > 1 && (x_stride < 0 || x_stride > (1 << 24))) || (n > 1 && (w_stride < k || w_stride > (1 << 24))))
    return fail(TG_EINVAL, "tg_linear_i8: row strides (x %lld, w %lld) out of range", (long long)x_stride, (long long)w_stride);
  if (rows > 1 && (out_stride < n || out_stride > (1 << 24))) return fail(TG_EINVAL, "tg_linear_i8: the output's row stride %lld must be n .. 2^24", (long long)out_stride);
  if (n > (1 << 22) || rows > ((int64_t)1 << 34)) return fail(TG_EINVAL, "tg_linear_i8: n = %lld or rows = %lld too large", (long long)n, (long long)rows);
  if (!out || !w_scale || (k && (!x || !w))) return fail(TG_EINVAL, "tg_linear_i8: null pointer");
  const int os = type_size(out_type);
  if ((uintptr_t)out % os || (uintptr_t)w_scale % 4 || (uintptr_t)x_scale % 4 || (uintptr_t)bias % 4)
    return fail(TG_EINVAL, "tg_linear_i8: out / w_scale / x_scale / bias not aligned to their elements");
  if (rows == 1) { x_stride = k; out_stride = n; }
  if (n == 1) w_stride = k;
  if (k == 0) x_stride = w_stride = 0;  // (no operand: strides of empty rows must not span bytes that are not there)
  const int64_t no = span(rows, n, out_stride, os), nx = k ? span(rows, k, x_stride, 1) : 0, nw = k ? span(n, k, w_stride, 1) : 0;
  if (no < 0 || nx < 0 || nw < 0) return fail(TG_EINVAL, "tg_linear_i8: an array of more than 2^47 bytes");
  if ((k && (overlap(out, no, x, nx) || overlap(out, no, w, nw))) || overlap(out, no, w_scale, 4 * n) ||
      overlap(out, no, x_scale, 4 * rows) || overlap(out, no, bias, 4 * n))
    return fail(TG_EINVAL, "tg_linear_i8: the output overlaps an input");
  ON_DEVICE("tg_linear_i8", device);
  LinearArgs a{(const uint8_t*)x, w, w_scale, x_scale, bias, out, rows, k, n, x_stride, w_stride, out_stride, relu != 0};
  return launched("tg_linear_i8", by_float(out_type, [&](auto o) {
    using OT = decltype(o);
    return x_type == kU8 ? linear_launch<OT, true>(a, (hipStream_t)stream) : linear_launch<OT, false>(a, (hipStream_t)stream);
  }));
}

int tg_quantize_i8(int device, void* stream, const void* x, int x_type, int64_t rows, int64_t k, int64_t x_stride, int8_t* q, int64_t q_stride,
                   float* scale) {
  if (!is_float(x_type)) return fail(TG_EINVAL, "tg_quantize_i8: x must be f32, f16 or bf16, got type %d", x_type);
  if (rows < 0 || k < 0 || rows > kMaxGroups || k > (1 << 30)) return fail(TG_EINVAL, "tg_quantize_i8: bad sizes (rows %lld, k %lld)", (long long)rows, (long long)k);
  if (rows == 0) return TG_OK;
  if (rows > 1 && (x_stride < 0 || x_stride > (1 << 30) || q_stride < k || q_stride > (1 << 30)))
    return fail(TG_EINVAL, "tg_quantize_i8: row strides (x %lld, q %lld) out of range", (long long)x_stride, (long long)q_stride);
  if (!scale || (k && (!x || !q))) return fail(TG_EINVAL, "tg_quantize_i8: null pointer");
  const int size = type_size(x_type);
  if ((uintptr_t)x % size || (uintptr_t)scale % 4) return fail(TG_EINVAL, "tg_quantize_i8: x / scale not aligned to their elements");
  if (rows == 1) { x_stride = k; q_stride = k; }
  if (k) {
    const int64_t nx = span(rows, k, x_stride, size), nq = span(rows, k, q_stride, 1);
    if (nx < 0 || nq < 0) return fail(TG_EINVAL, "tg_quantize_i8: an array of more than 2^47 bytes");
    if (overlap(q, nq, x, nx) || overlap(scale, 4 * rows, x, nx) || overlap(scale, 4 * rows, q, nq))
      return fail(TG_EINVAL, "tg_quantize_i8: the outputs overlap each other or the input");
  }
  ON_DEVICE("tg_quantize_i8", device);
  return launched("tg_quantize_i8", by_float(x_type, [&](auto e) {
    using T = decltype(e);
    const int64_t vec = kQVec<T>;
    // rows in as few registers as they need: four or sixteen lanes a row, then a wave, then a workgroup
    const auto run = [&](auto kernel, int rpb) {
      const int64_t most = max_blocks(256) * rpb;
      for (int64_t r = 0; r < rows; r += most) {
        const int64_t m = rows - r < most ? rows - r : most;
        const hipError_t err = launch(kernel, dim3((unsigned)((m + rpb - 1) / rpb)), dim3(256), 0, (hipStream_t)stream, (const T*)x + r * x_stride, m, k, x_stride,
                                      q + r * q_stride, q_stride, scale + r);
        if (err != hipSuccess) return err;
      }
      return hipSuccess;
    };
    if (k <= 4 * vec) return run(quantize_kernel<T, 4, 1>, 64);
    if (k <= 8 * vec) return run(quantize_kernel<T, 4, 2>, 64);
    if (k <= 16 * vec) return run(quantize_kernel<T, 16, 1>, 16);
    if (k <= 32 * vec) return run(quantize_kernel<T, 16, 2>, 16);
    if (k <= 64 * vec) return run(quantize_kernel<T, 16, 4>, 16);
    if (k <= 128 * vec) return run(quantize_kernel<T, 64, 2>, 4);
    if (k <= 256 * vec) return run(quantize_kernel<T, 64, 4>, 4);
    if (k <= 512 * vec) return run(quantize_kernel<T, 256, 2>, 1);
    if (k <= 1024 * vec) return run(quantize_kernel<T, 256, 4>, 1);
    return run(quantize_kernel<T, 256, 8>, 1);
  }));
}

int64_t tg_beam_select_workspace(int64_t groups, int64_t beams_in, int64_t vocab, int64_t beams_out) {
  if (groups < 0 || beams_in < 0 || vocab < 0 || beams_out < 0) return fail(TG_EINVAL, "tg_beam_select_workspace: negative size");
  if (groups > kMaxGroups || beams_in > TG_OPS_MAX_BEAMS || beams_out > TG_OPS_MAX_BEAMS || vocab > TG_OPS_MAX_VOCAB)
    return fail(TG_EINVAL, "tg_beam_select_workspace: %lld groups, %lld beams in, %lld out, %lld entries: up to %lld, %d, %d, %d are supported", (long long)groups,
                (long long)beams_in, (long long)beams_out, (long long)vocab, (long long)kMaxGroups, TG_OPS_MAX_BEAMS, TG_OPS_MAX_BEAMS, TG_OPS_MAX_VOCAB);
  if (groups == 0 || beams_in == 0 || vocab == 0) return 0;
  const SelectPlan p = select_plan(groups, beams_in, vocab);
  return p.small ? 0 : groups * beams_in * p.chunks * select_part_bytes((int)beams_out);
}

int tg_beam_select(int device, void* stream, const void* logits, int type, int64_t groups, int64_t beams_in, int64_t vocab, int64_t lg,
                   int64_t lk, const float* scores, const uint8_t* mask, int64_t mg, int64_t mk, const uint8_t* finished, int pad,
                   int normalize, int64_t beams_out, float* out_scores, int32_t* parents, int32_t* tokens, void* workspace,
                   int64_t workspace_bytes) {
  if (!is_float(type)) return fail(TG_EINVAL, "tg_beam_select: logits must be f32, f16 or bf16, got type %d", type);
  if (groups < 0 || groups > kMaxGroups) return fail(TG_EINVAL, "tg_beam_select: %lld groups", (long long)groups);
  if (beams_in < 1 || beams_in > TG_OPS_MAX_BEAMS || beams_out < 1 || beams_out > TG_OPS_MAX_BEAMS)
    return fail(TG_EINVAL, "tg_beam_select: %lld beams in, %lld out: 1 .. %d are supported", (long long)beams_in, (long long)beams_out, TG_OPS_MAX_BEAMS);
  if (vocab < 1 || vocab > TG_OPS_MAX_VOCAB) return fail(TG_EINVAL, "tg_beam_select: %lld entries: 1 .. %d are supported", (long long)vocab, TG_OPS_MAX_VOCAB);
  if (finished && (pad < 0 || pad >= vocab)) return fail(TG_EINVAL, "tg_beam_select: pad %d outside the %lld entries", pad, (long long)vocab);
  if (groups == 0) return TG_OK;
  if (lg < 0 || lk < 0 || lg > kMost || lk > kMost / 64 || (mask && (mg < 0 || mk < 0 || mg > kMost || mk > kMost / 64)))
    return fail(TG_EINVAL, "tg_beam_select: negative or too large strides");
  if (!logits || !scores || !out_scores || !parents || !tokens) return fail(TG_EINVAL, "tg_beam_select: null pointer");
  if ((uintptr_t)logits % type_size(type) || (uintptr_t)scores % 4 || (uintptr_t)out_scores % 4 || (uintptr_t)parents % 4 || (uintptr_t)tokens % 4)
    return fail(TG_EINVAL, "tg_beam_select: an array is not aligned to its elements");
  const SelectPlan p = select_plan(groups, beams_in, vocab);
  const int64_t need = tg_beam_select_workspace(groups, beams_in, vocab, beams_out);
  if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
    return fail(TG_EINVAL, "tg_beam_select: a 16-byte aligned workspace of %lld bytes is needed, got %lld", (long long)need, (long long)workspace_bytes);
  {
    const int64_t no = 4 * groups * beams_out, ni = 4 * groups * beams_in;
    const int64_t nl = span(beams_in, vocab, lk, type_size(type), groups, lg), nm = mask ? span(beams_in, vocab, mk, 1, groups, mg) : 0;
    if (nl < 0 || nm < 0) return fail(TG_EINVAL, "tg_beam_select: an array of more than 2^47 bytes");
    const void* outs[3] = {out_scores, parents, tokens};
    for (int i = 0; i < 3; ++i) {
      if (overlap(outs[i], no, logits, nl) || overlap(outs[i], no, scores, ni) || (mask && overlap(outs[i], no, mask, nm)) ||
          overlap(outs[i], no, finished, ni / 4) || overlap(outs[i], no, outs[(i + 1) % 3], no) || (need && overlap(outs[i], no, workspace, need)))
        return fail(TG_EINVAL, "tg_beam_select: the outputs overlap each other or an input");
    }
    if (need && (overlap(workspace, need, logits, nl) || overlap(workspace, need, scores, ni) || (mask && overlap(workspace, need, mask, nm)) ||
                 overlap(workspace, need, finished, ni / 4)))
      return fail(TG_EINVAL, "tg_beam_select: the workspace overlaps an input");
  }
  ON_DEVICE("tg_beam_select", device);
  const int merge_threads = 64 * (!normalize ? 1 : beams_in < 16 ? (int)beams_in : 16);
  int64_t most = max_blocks(256) * 4;  // groups of one launch
  if (!p.small) most = std::min(max_blocks(256) / (beams_in * p.chunks), max_blocks(merge_threads));
  // (some groups of it, for one launch of each kernel)
  const auto run = [&](auto e, int64_t g, int64_t groups) {
    using T = decltype(e);
    const SelectArgs a{(const T*)logits + g * lg, scores + g * beams_in, mask ? mask + g * mg : nullptr, finished ? finished + g * beams_in : nullptr,
                       out_scores + g * beams_out, parents + g * beams_out, tokens + g * beams_out, lg, lk, mg, mk, groups, (int)beams_in, (int)vocab,
                       (int)beams_out, pad, normalize != 0};
    const hipStream_t st = (hipStream_t)stream;
    if (p.small) {
      const dim3 grid((unsigned)((groups + 3) / 4));
      if (p.per_lane <= 2) return launch(select_small_kernel<T, 2>, grid, dim3(256), 0, st, a, p.shift);
      if (p.per_lane <= 5) return launch(select_small_kernel<T, 5>, grid, dim3(256), 0, st, a, p.shift);
      if (p.per_lane <= 8) return launch(select_small_kernel<T, 8>, grid, dim3(256), 0, st, a, p.shift);
      return launch(select_small_kernel<T, 16>, grid, dim3(256), 0, st, a, p.shift);
    }
    const dim3 grid((unsigned)(groups * beams_in * p.chunks));
    uint8_t* ws = (uint8_t*)workspace + g * beams_in * p.chunks * select_part_bytes((int)beams_out);
    const auto chunks = [&](auto kernel) { return launch(kernel, grid, dim3(256), 0, st, a, p.chunks, ws); };
    const hipError_t err = p.e == 8 ? chunks(select_chunk_kernel<T, 8>) : p.e == 16 ? chunks(select_chunk_kernel<T, 16>) : chunks(select_chunk_kernel<T, 32>);
    return err != hipSuccess ? err : launch(select_merge_kernel, dim3((unsigned)groups), dim3(merge_threads), 0, st, a, p.chunks, (const uint8_t*)ws);
  };
  return launched("tg_beam_select", by_float(type, [&](auto e) {
    for (int64_t g = 0; g < groups; g += most) {
      const hipError_t err = run(e, g, groups - g < most ? groups - g : most);
      if (err != hipSuccess) return err;
    }
    return hipSuccess;
  }));
}

int tg_beam_reorder(int device, void* stream, int n, const void* const* src, void* const* dst, const int64_t* row_bytes,
                    const int64_t* src_stride, const int64_t* dst_stride, int64_t groups, int64_t beams_in, int64_t beams_out,
                    const int32_t* parents) {
  if (n < 0 || n > TG_OPS_MAX_STATES) return fail(TG_EINVAL, "tg_beam_reorder: %d arrays: up to %d go into one call", n, TG_OPS_MAX_STATES);
  if (groups < 0 || groups > kMaxGroups) return fail(TG_EINVAL, "tg_beam_reorder: %lld groups", (long long)groups);
  if (beams_in < 1 || beams_in > TG_OPS_MAX_BEAMS || beams_out < 1 || beams_out > TG_OPS_MAX_BEAMS)
    return fail(TG_EINVAL, "tg_beam_reorder: %lld beams in, %lld out: 1 .. %d are supported", (long long)beams_in, (long long)beams_out, TG_OPS_MAX_BEAMS);
  if (n == 0 || groups == 0) return TG_OK;
  if (!src || !dst || !row_bytes || !src_stride || !dst_stride || !parents) return fail(TG_EINVAL, "tg_beam_reorder: null pointer");
  if ((uintptr_t)parents % 4) return fail(TG_EINVAL, "tg_beam_reorder: parents not aligned");
  static_assert(2 * TG_OPS_MAX_STATES <= kReorderMax, "a row's whole units and its rest");
  ReorderArgs p;
  p.n = 0;
  p.items = 0;
  const int64_t rin = groups * beams_in, rout = groups * beams_out;
  for (int i = 0; i < n; ++i) {
    const int64_t rb = row_bytes[i], ss = src_stride[i], ds = dst_stride[i];
    if (rb < 0 || rb > kMost || ss < rb || ds < rb || ss > kMost / 64 || ds > kMost / 64)
      return fail(TG_EINVAL, "tg_beam_reorder: array %d: rows of %lld bytes at strides %lld / %lld", i, (long long)rb, (long long)ss, (long long)ds);
    if (rb && (span(rin, rb, ss, 1) < 0 || span(rout, rb, ds, 1) < 0)) return fail(TG_EINVAL, "tg_beam_reorder: array %d: more than 2^47 bytes", i);
  }
  bool in_place = false, first = true;  // (by the first array that has bytes: an empty one may stand at any address)
  for (int i = 0; i < n; ++i) {
    const int64_t rb = row_bytes[i], ss = src_stride[i], ds = dst_stride[i];
    if (rb == 0) continue;
    if (!src[i] || !dst[i]) return fail(TG_EINVAL, "tg_beam_reorder: array %d is null", i);
    if (first) in_place = dst[i] == src[i];
    first = false;
    const int64_t nd = span(rout, rb, ds, 1);
    if (overlap(dst[i], nd, parents, 4 * rout)) return fail(TG_EINVAL, "tg_beam_reorder: array %d overlaps the parents", i);
    if ((dst[i] == src[i]) != in_place) return fail(TG_EINVAL, "tg_beam_reorder: some arrays in place and some not");
    if (in_place && (ss != ds || beams_in != beams_out)) return fail(TG_EINVAL, "tg_beam_reorder: array %d: in place needs equal strides and beams", i);
    for (int j = 0; j < n; ++j) {
      if (row_bytes[j] == 0 || (in_place && j == i)) continue;
      if (overlap(dst[i], nd, src[j], span(rin, row_bytes[j], src_stride[j], 1)) ||
          (j != i && overlap(dst[i], nd, dst[j], span(rout, row_bytes[j], dst_stride[j], 1))))
        return fail(TG_EINVAL, "tg_beam_reorder: arrays %d and %d overlap", i, j);
    }
    const int64_t most = 64 * kReorderReg / beams_out;  // columns of an item of one group
    // Units of 16 bytes; what is left of a row goes as one more unit that overlaps the last where an item holds whole rows (nobody else
    // reads those bytes then), else as an array of its own in the largest units that divide it.
    const bool over = rb >= 16 && rb % 16 && (rb + 15) / 16 <= most;
    const int64_t whole = over ? rb : rb >= 16 ? rb & ~(int64_t)15 : 0;
    for (const int64_t part : {whole, rb - whole}) {
      if (part == 0) continue;
      const int64_t at = part == whole ? 0 : whole;
      ReorderArray& a = p.a[p.n];
      a.src = (const uint8_t*)src[i] + at;
      a.dst = (uint8_t*)dst[i] + at;
      a.src_stride = ss;
      a.dst_stride = ds;
      a.shift = over ? 4 : __builtin_ctzll((uint64_t)part | 16);
      a.units = (part + (1 << a.shift) - 1) >> a.shift;
      a.last = part - (1 << a.shift);
      a.cb = (int)(a.units < most ? a.units : most);
      a.gp = a.cb < a.units ? 1 : (int)(64 * kReorderReg / (beams_out * a.cb));
      a.mul_cb = ((1u << 21) + a.cb - 1) / a.cb;
      a.mul_out = ((1u << 21) + (uint32_t)beams_out - 1) / (uint32_t)beams_out;
      const int64_t blocks = (a.units + a.cb - 1) / a.cb, sets = (groups + a.gp - 1) / a.gp;
      if (blocks > kMaxGroups || sets > (kMaxGroups - p.items) / blocks) return fail(TG_EINVAL, "tg_beam_reorder: too much in one call (array %d)", i);
      a.blocks = (uint32_t)blocks;
      p.first[p.n] = p.items;
      p.items += (uint32_t)(blocks * sets);
      ++p.n;
    }
  }
  if (p.n == 0) return TG_OK;
  for (int i = p.n; i < kReorderMax; ++i) p.first[i] = 0xFFFFFFFFu;
  p.parents = parents;
  p.groups = groups;
  p.kin = (int)beams_in;
  p.kout = (int)beams_out;
  p.in_place = in_place;
  ON_DEVICE("tg_beam_reorder", device);
  hipError_t err = hipSuccess;
  const uint32_t most = (uint32_t)(4 * max_blocks(256));  // items of one launch
  for (p.base = 0; err == hipSuccess && p.base < p.items; p.base += most)
    err = launch(reorder_kernel, dim3((std::min(p.items - p.base, most) + 3) / 4), dim3(256), 0, (hipStream_t)stream, p);
  return launched("tg_beam_reorder", err);
}

int tg_beam_advance(int device, void* stream, int64_t groups, int64_t beams, const int32_t* parents, const int32_t* tokens,
                    const float* gain_in, float* gain_out, int32_t* actions) {
  if (groups < 0 || groups > kMaxGroups || beams < 1 || beams > TG_OPS_MAX_BEAMS)
    return fail(TG_EINVAL, "tg_beam_advance: %lld groups of %lld beams", (long long)groups, (long long)beams);
  const int64_t n = groups * beams;
  if (n > 256 * max_blocks(256)) return fail(TG_EINVAL, "tg_beam_advance: %lld groups of %lld beams: up to %lld environments are supported", (long long)groups, (long long)beams, (long long)(256 * max_blocks(256)));
  if (n == 0) return TG_OK;
  if (!parents || !tokens || !gain_in || !gain_out || !actions) return fail(TG_EINVAL, "tg_beam_advance: null pointer");
  if (overlap(gain_out, 4 * n, gain_in, 4 * n)) return fail(TG_EINVAL, "tg_beam_advance: gain_out overlaps gain_in");
  ON_DEVICE("tg_beam_advance", device);
  return launched("tg_beam_advance", launch(advance_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, (hipStream_t)stream, parents, tokens, gain_in, gain_out, actions, n, (int)beams));
}

int tg_beam_collect(int device, void* stream, int64_t n, const tg_step_out* out, float* gain) {
  if (n < 0 || n > kMaxGroups) return fail(TG_EINVAL, "tg_beam_collect: %lld environments", (long long)n);
  if (n == 0) return TG_OK;
  if (!out || !gain) return fail(TG_EINVAL, "tg_beam_collect: null pointer");
  ON_DEVICE("tg_beam_collect", device);
  return launched("tg_beam_collect", launch(collect_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, (hipStream_t)stream, out, gain, n));
}

}  // extern "C"
