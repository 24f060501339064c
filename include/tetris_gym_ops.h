/*
 * tetris_gym_ops.h — C ABI of the operators between the engine's observations and its actions (libtetris_gym_hip.so):
 * the product of 8-bit observations or quantised activations with 8-bit weights, the selection of a beam search under a
 * legal mask, and the reordering of the states that follow their beams.
 *
 * Every pointer is DEVICE memory of `device` unless it says host.  Calls are asynchronous on `stream` (a hipStream_t; NULL =
 * the default stream), allocate nothing, keep nothing, and can be captured into a graph.  They return 0 or a TG_E* code of
 * tetris_gym_hip.h; the message of the calling thread's last failure is tg_ops_last_error() (of the calls that take a handle it is
 * tg_last_error(handle) too).  The caller's current device is left as it was.  Strides count elements; the innermost axis is contiguous.
 * No array spans more than 2^47 bytes.
 */
#ifndef TETRIS_GYM_OPS_H
#define TETRIS_GYM_OPS_H

#include <stddef.h>
#include <stdint.h>

#include "tetris_gym_hip.h" /* tg_handle, TG_E* */

#ifdef __cplusplus
extern "C" {
#endif

/* element types */
#define TG_T_U8 0
#define TG_T_I8 1
#define TG_T_F32 2
#define TG_T_F16 3
#define TG_T_BF16 4

#define TG_OPS_MAX_K 65536      /* longest sum of tg_linear_i8 (255 * 128 * 65536 < 2^31) */
#define TG_OPS_MAX_BEAMS 64     /* beams of a group, in and out */
#define TG_OPS_MAX_VOCAB (1 << 20) /* entries of tg_beam_select */
#define TG_OPS_MAX_STATES 24    /* arrays of one tg_beam_reorder */

const char* tg_ops_last_error(void);

/* out[m][n] = act((sum_k x[m][k] * w[n][k]) * (x_scale[m] * w_scale[n]) + bias[n]): the sum in 32-bit integers (exact), the rest in
 * float32, one rounding to the output's type.  x: u8 or i8 [rows][k] (x_stride; any alignment: observations of 13 or 200 bytes; row strides up to 2^24),
 * w: i8 [n][k] (row strides k .. 2^24), w_scale f32[n], x_scale f32[rows] or NULL (1), bias f32[n] or NULL, relu: act = max(., 0), else identity.
 * out: f32 / f16 / bf16 [rows][n] (out_stride).  rows or n = 0 does nothing; k = 0 gives act(bias).  out must not overlap an input.
 * Up to 2^34 rows, 2^22 columns n. */
int tg_linear_i8(int device, void* stream, const void* x, int x_type, int64_t rows, int64_t k, int64_t x_stride, const int8_t* w, int64_t n,
                 int64_t w_stride, const float* w_scale, const float* x_scale, const float* bias, int relu, void* out, int out_type,
                 int64_t out_stride);

/* scale[m] = max(max_k |x[m][k]| / 127, 2^-126) (float32), q[m][k] = x / scale rounded half to even (of the real quotient): a row times
 * its scale is the row to half a step.  A row with a NaN or an infinity gets scale NaN and q 0, so that a product made from it is
 * NaN too.  x: f32 / f16 / bf16 [rows][k] (x_stride 0 .. 2^30); q: i8 [rows][k] (q_stride k .. 2^30); scale f32[rows].
 * Fewer than 2^31 rows, k up to 2^30. */
int tg_quantize_i8(int device, void* stream, const void* x, int x_type, int64_t rows, int64_t k, int64_t x_stride, int8_t* q, int64_t q_stride,
                   float* scale);

/* One step of a beam search for `groups` independent searches.  Beam j of group g holds scores[g * beams_in + j] and offers for entry v
 *   c = scores + logits[v] - L,   L = normalize ? log sum exp over the beam's allowed entries : 0
 * where mask (u8, nonzero = allowed; NULL = all) allows v.  A beam whose finished byte is set offers the single candidate (pad, scores)
 * instead.  A candidate whose c is -inf or NaN does not exist (a dead beam: scores = -inf); what stands at a masked place is
 * never read into a result.  The beams_out best of the group by c come out in descending order: out_scores f32, parents i32 (0 ..
 * beams_in - 1), tokens i32 (0 .. vocab - 1); equal ones by beam, then by entry; within one beam entries rank by their logit.  Where
 * there are fewer: score -inf, parent -1, token -1.  logits: f32 / f16 / bf16 [groups][beams_in][vocab] (strides lg, lk; lk = 0 or
 * lg = 0 broadcasts), mask likewise (mg, mk), scores / finished [groups][beams_in] and the outputs [groups][beams_out] contiguous.
 * c is held and ranked in 64 bits with L good to 1e-12, and rows of logits that differ by a constant get the same log-probabilities (a single
 * allowed entry 0): only scores nearer than that to each other may come out in another order than their exact values.
 * workspace: tg_beam_select_workspace bytes (0 for small searches, TG_EINVAL beyond the limits above), 16-byte aligned, not shared by
 * calls that may run at the same time and apart from every other array.  Fewer than 2^31 groups. */
int64_t tg_beam_select_workspace(int64_t groups, int64_t beams_in, int64_t vocab, int64_t beams_out);
int tg_beam_select(int device, void* stream, const void* logits, int type, int64_t groups, int64_t beams_in, int64_t vocab, int64_t lg,
                   int64_t lk, const float* scores, const uint8_t* mask, int64_t mg, int64_t mk, const uint8_t* finished, int pad,
                   int normalize, int64_t beams_out, float* out_scores, int32_t* parents, int32_t* tokens, void* workspace,
                   int64_t workspace_bytes);

/* Rows that follow their beams, for n (<= TG_OPS_MAX_STATES) arrays in one launch: dst[a][g][j] = src[a][g][parents[g][j]], rows of
 * row_bytes[a] bytes at src_stride[a] / dst_stride[a] bytes, parents i32 [groups][beams_out].  A parent outside 0 .. beams_in - 1 (the
 * -1 of tg_beam_select) leaves the row as it was.  dst[a] == src[a] with the same stride and beams_in == beams_out reorders in place;
 * any other overlap is refused.  Strides up to 2^34, fewer than 2^31 groups.  src, dst, row_bytes, src_stride, dst_stride are HOST arrays of n entries. */
int tg_beam_reorder(int device, void* stream, int n, const void* const* src, void* const* dst, const int64_t* row_bytes,
                    const int64_t* src_stride, const int64_t* dst_stride, int64_t groups, int64_t beams_in, int64_t beams_out,
                    const int32_t* parents);

/* The same for an engine: env g * beams + j becomes a copy of env g * beams + parents[g][j] in every respect (board, record, generator,
 * observation, last outputs, episode statistics), in place, asynchronous on the handle's stream.  batch must be a multiple of beams
 * and every env must have been reset (NUMPY rules).  What is computed on demand stays as it was: the legal mask, the features, and
 * actions drawn by tg_grouped_sample, which belong to the states they were drawn for. */
int tg_reorder_beams(tg_handle* h, const int32_t* parents, int beams);

/* The bookkeeping of a search between tg_beam_select and a transition, for groups * beams environments: gain_out = gain_in of the parent
 * and actions = the token where a beam has a parent; gain_out = -inf (a dead beam) and action 0 where it has none.  gain_out must not
 * overlap gain_in.  Fewer than 2^32 - 256 environments. */
int tg_beam_advance(int device, void* stream, int64_t groups, int64_t beams, const int32_t* parents, const int32_t* tokens,
                    const float* gain_in, float* gain_out, int32_t* actions);

/* ... and behind the transition: gain += reward, or -inf where the game has ended (n environments). */
int tg_beam_collect(int device, void* stream, int64_t n, const tg_step_out* out, float* gain);

/* The handle's stream (a hipStream_t), for calls above that shall run in order with the handle's own.  (tg_config.streams > 1 spreads
 * transitions over further streams, which this call and every other one on the handle join: ask again behind a transition.) */
int tg_stream(tg_handle* h, void** stream);

#ifdef __cplusplus
}
#endif
#endif
