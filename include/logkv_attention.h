/*
 * C ABI of the read side of the SemanticLogKV cache: mid-anchor attention plan,
 * packing and slot attention over [merged slots | exact pool | recent window |
 * current tokens].  Same conventions as logkv_b200.h: caller-owned device
 * memory in the reference's layouts, work enqueued on the caller's stream, no
 * allocation, no host synchronization, 0 / negative LOGKV_E_* / CUDA error.
 */
#ifndef LOGKV_ATTENTION_H
#define LOGKV_ATTENTION_H

#include "logkv_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Attention plan of one layer.  cap = clusters * levels * slots.  The first block
 * is the reference's plan (LogStructuredKVCache._semantic_mid_attention_plan,
 * litgpt/log_kv_cache.py:5979-6007): per (b, g) lane the occupied ladder entries,
 * cluster-major with the top level first, their mid anchors
 * floor((2 sum_wp + ww) / (2 ww)), ww = max(trunc(w), 1), and valid = w > 0.
 * Entries past a lane's width are 0 / 0 / false, which is what the reference's
 * [B, G, width_max] tensors hold there.  The second block is the same plan with
 * the invalid entries dropped, and the valid exact-pool rows per batch row.
 */
typedef struct logkv_plan {
  int64_t* idx;        /* [B,G,cap] physical entry (c * L + level) * B' + slot     */
  int64_t* anchor;     /* [B,G,cap]                                               */
  uint8_t* valid;      /* [B,G,cap]                                               */
  int32_t* width;      /* [B,G] occupied entries per lane                         */
  int32_t* width_max;  /* [1]                                                     */
  int32_t* vslot;      /* [B,G,cap] physical entries of valid slots, plan order    */
  int64_t* vanchor;    /* [B,G,cap] their anchors                                 */
  int32_t* nvalid;     /* [B,G]                                                   */
  int32_t* exact_rows; /* [B,P] valid rows among the first alpha_count pool rows  */
  int32_t* nexact;     /* [B]                                                     */
} logkv_plan_t;

/* LitGPT RoPE tables (cos_cache / sin_cache of the cache, litgpt/log_kv_position.py:74-101). */
typedef struct logkv_rope {
  const void* cos;  /* [rows, rope_n] */
  const void* sin;  /* [rows, rope_n] */
  int32_t rows;     /* positions in the tables; a larger anchor sets status bit 16 and is clamped */
  int32_t rope_n;   /* rotated leading features: even, <= dim (0 = no rotation) */
  int32_t dtype;    /* LOGKV_DTYPE_F32 or LOGKV_DTYPE_BF16 */
} logkv_rope_t;

/*
 * Packed frozen prefix for attention, rebuilt once per flush: per lane the valid
 * merged slots (plan order, keys rotated at their mid anchors) followed by the
 * valid exact-pool rows (keys rotated at alpha_pos), values as stored, and the
 * mass term log(max(w, 1)) rounded to the storage dtype (0 for exact rows).
 */
typedef struct logkv_prefix {
  void* k;           /* [B,G,capacity,D] storage dtype */
  void* v;           /* [B,G,capacity,D]               */
  float* mass;       /* [B,G,capacity]                 */
  int32_t* length;   /* [B,G]                          */
  int32_t capacity;  /* >= clusters * levels * slots + exact */
} logkv_prefix_t;

/* Plan of the current ladder state (reads level_count, level_w, level_sum_wp, alpha_valid, alpha_count). */
LOGKV_API int logkv_attention_plan(const logkv_layout_t* layout, const logkv_state_t* state,
                                   const logkv_plan_t* plan, void* stream);

/*
 * Pack the frozen prefix from a plan.  Replaces the pooled and exact parts of
 * the reference's packer (_pack_torch, litgpt/log_kv_pack.py:27-72) and the
 * reference's decode workspace reuse (_mid_chunk_attention, log_kv_cache.py:6770-6799).
 * `status` (device int32, may be NULL) gets bit 16 when an anchor is outside the tables.
 */
LOGKV_API int logkv_pack_prefix(const logkv_layout_t* layout, const logkv_state_t* state,
                                const logkv_plan_t* plan, const logkv_rope_t* rope,
                                const logkv_prefix_t* prefix, int32_t* status, void* stream);

/*
 * The reference's packed K/V for SDPA ([B,G,length,dim], dim >= D + 1), bit for bit
 * (log_kv_pack.pack_mid_kv with the torch backend, litgpt/log_kv_pack.py:27-72 and
 * :114-131): length = width + alpha_count + recent_count + tokens; K column D holds
 * log(max(w,1)) / 0 / -10000 in the storage dtype.  `width` and `alpha_count` are the
 * host values the output was sized with.  skip_pooled != 0 leaves the first
 * width + alpha_count rows untouched; rows before width + alpha_count + recent_start
 * are left untouched likewise (the reference's decode-buffer reuse).  k_new/v_new
 * are contiguous [B,G,tokens,D].
 */
LOGKV_API int logkv_pack_mid(const logkv_layout_t* layout, const logkv_state_t* state, const logkv_plan_t* plan,
                             const logkv_rope_t* rope, int32_t width, int32_t alpha_count, int32_t recent_count,
                             const void* k_new, const void* v_new, int32_t tokens, void* out_k, void* out_v,
                             int32_t dim, int32_t skip_pooled, int32_t recent_start, int32_t* status, void* stream);

/*
 * Slot attention over [prefix | recent window | the call's `tokens` new tokens]
 * for the query tokens [q_offset, q_offset + q_tokens) of the call:
 *   out = softmax(scale * (q . k_s + qx * mass_s)) v_s,
 * with causal != 0 new token j visible to query token t iff j <= t (the reference's
 * lower-right causal tail), else every new token visible; every other slot visible.
 * Replaces log_kv_chunk_attention (litgpt/log_kv_cache.py:6802-6864 ->
 * _mid_chunk_attention :6770-6799 -> Flash SDPA over the packed inputs of
 * _slot_sdpa_inputs :6439-6464).  qx is the query's mass coordinate, 1/scale
 * rounded to the storage dtype.
 *
 * Kernels: bf16 caches use tensor cores, a split-K decode kernel for up to 16 query
 * rows per lane (heads / groups * q_tokens in {1, 2, 4, 8, 16}) and a chunk kernel for
 * more (heads / groups a power of two <= 8, head dim <= 128); float32 caches use
 * CUDA cores for 1, 2, 4 or 8 query rows per lane (longer chunks take several calls).
 */
typedef struct logkv_attention_args {
  const void* q;        /* [B,H,q_stride,D] storage dtype, post-RoPE */
  const void* k_new;    /* [B,G,tokens,D] post-RoPE                */
  const void* v_new;    /* [B,G,tokens,D]                          */
  void* out;            /* [B,H,q_stride,D] storage dtype; rows [q_offset, q_offset + q_tokens) written */
  int32_t heads;        /* H, a multiple of groups                 */
  int32_t tokens;       /* new tokens (>= 1)                       */
  int32_t q_offset;     /* first query token of this call          */
  int32_t q_tokens;     /* query tokens of this call               */
  int32_t recent_count; /* window rows [0, recent_count) are attended */
  int32_t causal;       /* 1: causal tail over the new tokens, 0: none */
  float scale;
  float qx;
  int32_t q_stride;     /* query / output rows per head: 0 = tokens; fewer (causal 0 only) when the queries
                           are the first of the new tokens, e.g. a decode step whose single query sees a
                           pending token and itself (litgpt/model.py:1219-1226, causal_tail=0) */
} logkv_attention_args_t;

/* Scratch bytes of logkv_attention (zero-fill it once when allocated; calls leave it reusable). */
LOGKV_API size_t logkv_attention_workspace_bytes(const logkv_layout_t* layout, int32_t heads, int32_t q_tokens,
                                                 int32_t prefix_capacity);

LOGKV_API int logkv_attention(const logkv_layout_t* layout, const logkv_state_t* state,
                              const logkv_prefix_t* prefix, const logkv_attention_args_t* args,
                              void* workspace, size_t workspace_bytes, void* stream);

/*
 * Attention of a tree of drafted tokens over the cache (speculative decoding; no reference
 * counterpart).  The drafted tokens are not committed: token t of a batch row attends over
 * [prefix | recent window | itself and its ancestors in the tree],
 *   out = softmax(scale * (q . k_s + qx * mass_s)) v_s,
 * where the ancestors of t are parents[t], parents[parents[t]], ...  parents[t] = -1: t follows the
 * last committed token; 0 <= parents[t] < t: t follows token parents[t]; -2: no token (rows of a
 * batch whose trees are smaller are padded so).  Any other value is treated as -2 and sets bit 18
 * of `status` (bit 17: a bounded wait expired, the output is not valid).  A token that is absent, or
 * whose chain of parents reaches an absent token, writes a zero output row and is seen by no token: its
 * K and V may hold anything.  A token whose V holds a NaN or an infinity makes the outputs of the tokens
 * that see it NaN, and only those.
 *
 * q is [B,H,tokens,D], k_new and v_new are [B,G,tokens,D] (post-RoPE, storage dtype) with the given
 * element strides of their batch, head and token axes; the head dim is contiguous and every row
 * 16-byte aligned.  out is [B,H,tokens,D], contiguous.  Any number of query heads per group;
 * tokens <= LOGKV_TREE_MAX_TOKENS.  Head dims: 16, 32, 64, 128 (and 256 for bf16 caches).
 */
#define LOGKV_TREE_MAX_TOKENS 256
typedef struct logkv_tree_args {
  const void* q;
  const void* k_new;
  const void* v_new;
  void* out;
  const void* parents;      /* [B, tokens] int32, or int64 with parents_wide   */
  int64_t q_strides[3];
  int64_t k_strides[3];
  int64_t v_strides[3];
  int64_t parents_stride;   /* elements between batch rows; 0: one tree for all */
  int32_t parents_wide;     /* 1: parents are int64                             */
  int32_t heads;            /* H, a multiple of groups                          */
  int32_t tokens;
  int32_t recent_count;     /* window rows [0, recent_count) are attended       */
  float scale;
  float qx;                 /* as logkv_attention_args_t                        */
  int32_t* status;          /* device int32 or NULL                             */
} logkv_tree_args_t;

/* Scratch bytes of logkv_tree_attention (no initialisation needed; 0: shape not supported).  The
 * scratch must not be shared by calls that may overlap on the GPU. */
LOGKV_API size_t logkv_tree_attention_workspace_bytes(const logkv_layout_t* layout, int32_t heads, int32_t tokens,
                                                      int32_t prefix_capacity);

LOGKV_API int logkv_tree_attention(const logkv_layout_t* layout, const logkv_state_t* state,
                                   const logkv_prefix_t* prefix, const logkv_tree_args_t* args, void* workspace,
                                   size_t workspace_bytes, void* stream);

/*
 * Attention of batch rows that share a long prefix (beams or samples of one prompt; no reference counterpart).
 * Rows r * beams .. r * beams + beams - 1 hold the same packed prefix and the same window rows [0, window_from):
 * those keys are read from the first of the rows, once per 128 of the request's query rows (bf16, head dim 64 or 128,
 * more than 16 rows) or once per 16 (otherwise); the window rows [window_from, recent_count)
 * and the new tokens are each row's own.  Otherwise the result of logkv_attention for q_tokens query tokens over
 * `tokens` new ones:
 *   out = softmax(scale * (q . k_s + qx * mass_s)) v_s,
 * with causal != 0 (tokens = q_tokens) new token j visible to query token t iff j <= t, else every new token
 * visible.  Rows are taken to agree as promised; nothing checks it.  A new token whose V holds a NaN or an infinity:
 * with causal != 0 and several query tokens the whole outputs of those that see it are NaN, and only those; in every
 * other call all query tokens of its batch row see it, and that feature of their outputs is not finite, the others are
 * as without it.
 *
 * q is [B,H,q_tokens,D], k_new and v_new are [B,G,tokens,D] (post-RoPE, storage dtype) with the given element
 * strides of their batch, head and token axes; the head dim is contiguous and every row 16-byte aligned.  out is
 * [B,H,q_tokens,D], contiguous.  Any number of query heads per group; B a multiple of beams; heads / groups *
 * q_tokens * beams <= 2^20.  Head dims: 16, 32, 64, 128 (and 256 for bf16 caches).  Bit 17 of `status`: a bounded
 * wait expired, the output is not valid.
 */
typedef struct logkv_shared_args {
  const void* q;
  const void* k_new;
  const void* v_new;
  void* out;
  int64_t q_strides[3];
  int64_t k_strides[3];
  int64_t v_strides[3];
  int32_t heads;            /* H, a multiple of groups                          */
  int32_t beams;            /* rows that share a prefix                         */
  int32_t q_tokens;
  int32_t tokens;           /* new tokens, >= q_tokens                          */
  int32_t recent_count;     /* window rows [0, recent_count) are attended       */
  int32_t window_from;      /* the first of them that are shared                */
  int32_t causal;
  float scale;
  float qx;                 /* as logkv_attention_args_t                        */
  int32_t* status;          /* device int32 or NULL                             */
} logkv_shared_args_t;

/* Scratch bytes of logkv_shared_attention with these sizes (its pointers are not looked at; no initialisation
 * needed; 0: shape not supported).  The scratch must not be shared by calls that may overlap on the GPU. */
LOGKV_API size_t logkv_shared_attention_workspace_bytes(const logkv_layout_t* layout, const logkv_shared_args_t* args,
                                                        int32_t prefix_capacity);

LOGKV_API int logkv_shared_attention(const logkv_layout_t* layout, const logkv_state_t* state,
                                     const logkv_prefix_t* prefix, const logkv_shared_args_t* args, void* workspace,
                                     size_t workspace_bytes, void* stream);

/*
 * Beam search: batch row b of the cache becomes the old row index[b], in place (no reference
 * counterpart).  index is [B] on the device, int32 or int64 (index_wide); any map is allowed (one row
 * taken over by several, swaps, cycles).  An entry outside [0, B) leaves its row as it is and sets bit
 * 19 of `status` (device int32, may be NULL); bit 20: a bounded wait for a copy expired.  Rows with
 * index[b] = b are not touched.
 *
 * window_from = -1: the whole rows: ladder, clusters, exact pool, span bookkeeping, s_h, the window's
 * rows [0, recent_count) and, when `prefix` is not NULL, the packed prefix.  K and V past a level's
 * count (zero in every row), prefix rows past their length and window rows from recent_count on
 * are not moved.
 * window_from >= 0: only the window's rows [window_from, recent_count), for a caller whose rows b and
 * index[b] hold the same ladder, pool and earlier window rows (hypotheses forked from one row since
 * the last flush).  batch <= LOGKV_REORDER_MAX_BATCH.
 */
#define LOGKV_REORDER_MAX_BATCH 512
LOGKV_API int logkv_reorder_batch(const logkv_layout_t* layout, const logkv_state_t* state,
                                  const logkv_prefix_t* prefix, int32_t recent_count, int32_t window_from,
                                  const void* index, int32_t index_wide, int32_t* status, void* stream);

/* The same for up to 30 contiguous [batch, ...] buffers of row_bytes bytes per row (a decoder's own
 * per-row state). */
typedef struct logkv_rows {
  void* base;
  int64_t row_bytes;
} logkv_rows_t;
LOGKV_API int logkv_reorder_rows(const logkv_rows_t* buffers, int32_t n, int32_t batch, const void* index,
                                 int32_t index_wide, int32_t* status, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* LOGKV_ATTENTION_H */
