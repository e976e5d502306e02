/*
 * C ABI of beam search's selection over beams and vocabulary.  Same conventions as logkv_b200.h:
 * caller-owned device memory, work enqueued on the caller's stream, no allocation, no host
 * synchronization, 0 / negative LOGKV_E_* / CUDA error.  No reference counterpart (the reference
 * decodes greedily or by sampling).
 */
#ifndef LOGKV_BEAM_H
#define LOGKV_BEAM_H

#include "logkv_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

#define LOGKV_BEAM_MAX_K 128
#define LOGKV_BEAM_MAX_WIDTH 256

/*
 * For each of `requests` requests the k best continuations (w, v) of its `width` beams by
 *   scores[w] + logits[w, v] - log sum_u exp(logits[w, u]),
 * best first, ties to the lower (w, v).  Per chosen continuation: its score (out_scores [N,k]
 * float32), the beam's row n * width + w (out_rows [N,k] int64) and v (out_tokens [N,k] int64).
 *
 * Scores are ordered as float64 sums order them, within a beam by the logits themselves (sums of
 * exponentials are float32 per thread, joined in float64, and taken again in float64 for beams whose scores
 * are too close for that); beams with the same logits tie exactly.
 *
 * A logit of -inf is never chosen.  A beam whose score is not finite, or that has a NaN or +inf logit
 * or no finite one, offers nothing.  Places without a continuation get score -inf, token 0 and row
 * n * width + min(place, width - 1).
 *
 * keep_places != 0 (k == width): the best continuation of a beam is written to the beam's own place,
 * the others to the places of beams without one, in order of score; so that, with out_rows as
 * logkv_reorder_batch's index, no row moves whose beam goes on.
 *
 * logits: float32 or bf16 (dtype), element strides n_stride and w_stride, vocabulary contiguous, any
 * alignment of the rows.  scores [N, width] float32, contiguous.
 */
typedef struct logkv_beam_args {
  const void* logits;
  const float* scores;
  float* out_scores;
  int64_t* out_rows;
  int64_t* out_tokens;
  int64_t n_stride, w_stride;
  int32_t dtype;        /* LOGKV_DTYPE_* of the logits                  */
  int32_t requests;     /* N >= 1                                       */
  int32_t width;        /* W in [1, LOGKV_BEAM_MAX_WIDTH]               */
  int32_t vocab;        /* V >= 1, W * V < 2^31                         */
  int32_t k;            /* 1 <= k <= min(W * V, LOGKV_BEAM_MAX_K)       */
  int32_t keep_places;
} logkv_beam_args_t;

/* Scratch bytes (no initialisation needed; 0: shape not supported).  Not to be shared by calls that
 * may overlap on the GPU. */
LOGKV_API size_t logkv_beam_workspace_bytes(int32_t requests, int32_t width, int32_t vocab, int32_t k);

LOGKV_API int logkv_beam_select(const logkv_beam_args_t* args, void* workspace, size_t workspace_bytes,
                                void* stream);

#ifdef __cplusplus
}
#endif

#endif /* LOGKV_BEAM_H */
