/*
 * C ABI of the adjustment of next-token logits in front of beam selection or sampling: penalties of repeated
 * tokens, biases and grammar masks.  Same conventions as logkv_b200.h: caller-owned device memory, work
 * enqueued on the caller's stream, no allocation, no host synchronization, 0 / negative LOGKV_E_* / CUDA
 * error.  No reference counterpart.
 */
#ifndef LOGKV_LOGITS_H
#define LOGKV_LOGITS_H

#include "logkv_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

#define LOGKV_LOGITS_MAX_BIAS 1024

/*
 * Row r of the [rows, vocab] logits, with c(v) the times that token v occurs in history[r, prompt:length] and
 * "seen" its occurring in history[r, :length]:
 *   y = x
 *   y = x > 0 ? x / repetition : x * repetition      where v is seen
 *   y = y - (frequency * c(v) + presence * [c(v) > 0])
 *   y = y + the sum of v's biases
 *   y = -inf                                         where the mask's bit of v is 0
 * in float32, rounded once; logits that nothing touches are copied bit by bit, and a masked one is -inf whatever
 * it was (NaN too).  A token's biases are summed in the order of their entries, so every result is the same from
 * run to run.  History and bias tokens outside [0, vocab) are passed over.
 *
 * Rows are (n, w) pairs: logits row r lies at (r / width) * n_stride + (r % width) * w_stride elements, `out`
 * likewise; vocabulary contiguous, any alignment.  `out` may be the logits themselves (same strides), and must not
 * overlap them otherwise.  Every other per-row array has a row stride in elements, 0 for one row for all.
 * lengths and prompts (int32, int64 with *_wide; NULL: `length`, `prompt`) are clamped to [0, history_len] and
 * [0, length].  repetition, presence, frequency: float32 per row, or NULL for the scalar; a repetition penalty must
 * be positive.  mask: bit v % 32 of word v / 32.
 */
typedef struct logkv_logits_args {
  const void* logits;
  void* out;
  int64_t n_stride, w_stride, out_n_stride, out_w_stride;
  const void* history;          /* NULL: no history */
  int64_t history_stride;
  const void* lengths;
  const void* prompts;
  const float* repetitions;
  const float* presences;
  const float* frequencies;
  const void* bias_tokens;      /* NULL: no biases */
  const float* bias_values;
  int64_t bias_tokens_stride, bias_values_stride;
  const int32_t* mask;          /* NULL: no mask */
  int64_t mask_stride;
  int32_t dtype;                /* LOGKV_DTYPE_* of logits and out */
  int32_t rows, width, vocab;
  int32_t history_len, length, prompt;
  int32_t history_wide, lengths_wide, prompts_wide, bias_wide;
  int32_t bias_count;           /* <= LOGKV_LOGITS_MAX_BIAS */
  float repetition, presence, frequency;
} logkv_logits_args_t;

LOGKV_API int logkv_adjust_logits(const logkv_logits_args_t* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* LOGKV_LOGITS_H */
