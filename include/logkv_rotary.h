/*
 * C ABI of rotary positions: queries and keys rotated with the cache's tables, and unrotated keys and
 * values brought into the cache's window (or any rows) with the rotation on the way.  Same conventions as
 * logkv_b200.h: caller-owned device memory, work enqueued on the caller's stream, no allocation, no host
 * synchronization, 0 / negative LOGKV_E_* / CUDA error.  No reference counterpart (the reference's model
 * rotates in PyTorch, litgpt/model.py, and its cache takes both forms of a key).
 */
#ifndef LOGKV_ROTARY_H
#define LOGKV_ROTARY_H

#include "logkv_attention.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * One tensor of a call: [batch, heads, tokens, dim] with the given element strides of its batch, head and
 * token axes, dim contiguous.  rotate = 1: `rotated` gets the rotated rows and `raw`, when not NULL, the
 * unrotated ones (in halves); rotate = 0: `raw` gets the rows as they are.  Outputs must not overlap inputs.
 */
typedef struct logkv_rotate_part {
  const void* src;
  void* rotated;
  void* raw;
  int64_t src_strides[3];
  int64_t rotated_strides[3];
  int64_t raw_strides[3];
  int32_t heads;
  int32_t rotate;
} logkv_rotate_part_t;

#define LOGKV_ROTATE_MAX_PARTS 3

/*
 * With n = rope_n, h = n / 2, c and s the table rows of the token's position:
 *   out[d] = x[d] c[d] - x[d + h] s[d]   (d < h),   x[d] c[d] + x[d - h] s[d]   (h <= d < n),   x[d]  (d >= n)
 * in float32, rounded once.  interleaved = 1: the rotated features come as pairs (2 i, 2 i + 1) and leave as
 * halves (i, i + h), which is how the cache rotates what it stores; a product of a query and a key does not
 * depend on the order.
 *
 * positions: int32, or int64 with positions_wide, element strides of batch and token; NULL: pos0 + token.
 * One outside the tables is rotated at the nearest table row and sets bit 16 of `status` (may be NULL).
 * positions_out (int64, may be NULL) gets the positions as given, row b at b * positions_out_stride;
 * ends / ends_out (uint8, may be NULL) are copied likewise.
 */
typedef struct logkv_rotate_args {
  logkv_rotate_part_t parts[LOGKV_ROTATE_MAX_PARTS];
  const void* positions;
  int64_t position_strides[2];
  int64_t pos0;
  int64_t* positions_out;
  int64_t positions_out_stride;
  const uint8_t* ends;
  uint8_t* ends_out;
  int64_t ends_stride;
  int64_t ends_out_stride;
  int32_t* status;
  int32_t positions_wide;
  int32_t n_parts;
  int32_t batch;
  int32_t tokens;
  int32_t dim;
  int32_t dtype;         /* LOGKV_DTYPE_* of every part */
  int32_t interleaved;
} logkv_rotate_args_t;

LOGKV_API int logkv_rotate(const logkv_rope_t* rope, const logkv_rotate_args_t* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* LOGKV_ROTARY_H */
