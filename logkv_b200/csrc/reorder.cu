// Batch rows of a cache taken over by the hypotheses that go on (C ABI in include/logkv_b200.h):
// row b of every state buffer becomes the old row index[b], in place.
//
// A buffer's batch row is `segs` segments of bytes; rows that stay are neither read nor written.
//
// Where every source row stays itself (beams that go on keep their places), a CTA copies up to 16 KB of
// one segment of one source to all rows that take it over, through registers.  Where a source row is
// itself taken over (swaps, chains, cycles), a CTA takes the same column of all sources into shared
// memory, waits, and then writes it; no other CTA touches that column, so no order among the rows and
// no second copy of the state is needed.
#include <algorithm>

#include "attn_common.cuh"

namespace logkv {

constexpr int32_t kStatusBadIndex = 1 << 19;
constexpr int kRowBuffers = 40;
constexpr int kReorderThreads = 256;
constexpr int kReorderBatch = 2048;
constexpr int kReorderStage = 32 * 1024;   // staged bytes per CTA (more above 512 source rows)
constexpr int kReorderTile = 16 * 1024;    // bytes a CTA copies at a time when nothing is staged

// Segment i of row b: base + b * stride + i * seg_stride, seg_bytes long.  With counts (of element
// size count_size, [B, segs]) only the first unit * max(count of the source, count of the row) bytes
// move: K and V past a level's count are zero in every row (a flush clears what it vacates), and
// prefix rows past the length are never read.
struct RowBuffer {
  char* base;
  const void* counts;
  long long stride, seg_stride;
  int segs, seg_bytes, unit;
  short count_size, width;   // width: bytes per access (16, 8, 4, 2 or 1)
};

struct RowArgs {
  RowBuffer buf[kRowBuffers];
  int n, B, wide;
  const void* index;
  int32_t* status;
};

__device__ __forceinline__ int row_count(const RowBuffer& r, int b, int seg) {
  const size_t at = (size_t)b * r.segs + seg;
  return r.count_size == 2 ? static_cast<const int16_t*>(r.counts)[at] : static_cast<const int32_t*>(r.counts)[at];
}

// Who takes over whom: sources (distinct, ascending) and, grouped by source, the rows that go on from them.
struct RowLists {
  short* src;     // [nsrc] source rows
  short* first;   // [nsrc + 1] their rows' places in dst
  short* dst;     // [nmov]
  int nsrc, nmov;
  bool chained;   // some source is itself taken over
};

__device__ __forceinline__ int source_of(const RowArgs& a, int b) {
  const long long v = a.wide ? static_cast<const long long*>(a.index)[b] : (long long)static_cast<const int32_t*>(a.index)[b];
  if (v >= 0 && v < a.B) return (int)v;
  if (blockIdx.x == 0) set_status(a.status, kStatusBadIndex);
  return b;
}

// By the whole block; from[B] and num[B] are scratch.
__device__ RowLists row_lists(const RowArgs& a, short* src, short* first, short* dst, short* from, int* num) {
  __shared__ int wsum[32];
  __shared__ int sh[3];
  RowLists r{src, first, dst, 0, 0, false};
  const int tid = threadIdx.x, B = a.B;
  if (B <= 32) {   // a warp, by ballots
    if (tid < 32) {
      const int s = tid < B ? source_of(a, tid) : tid;
      const bool moved = s != tid;
      const unsigned need = __reduce_or_sync(0xffffffffu, moved ? 1u << s : 0u);
      const unsigned mv = __ballot_sync(0xffffffffu, moved);
      int at = 0, n = 0;
      for (unsigned left = need; left; left &= left - 1) {
        const int x = __ffs(left) - 1;
        const unsigned who = __ballot_sync(0xffffffffu, moved && s == x);
        if (tid == 0) {
          src[n] = (short)x;
          first[n] = (short)at;
        }
        if (who >> tid & 1) dst[at + __popc(who & ((1u << tid) - 1))] = (short)tid;
        at += __popc(who);
        ++n;
      }
      if (tid == 0) {
        first[n] = (short)at;
        sh[0] = n;
        sh[1] = at;
        sh[2] = (need & mv) != 0;
      }
    }
    __syncthreads();
  } else {
    for (int b = tid; b < B; b += blockDim.x) {
      from[b] = (short)source_of(a, b);
      num[b] = 0;
    }
    if (tid == 0) sh[2] = 0;
    __syncthreads();
    for (int b = tid; b < B; b += blockDim.x)
      if (from[b] != b) atomicAdd(&num[from[b]], 1);
    __syncthreads();
    int nsrc = 0, nmov = 0;
    for (int b0 = 0; b0 < B; b0 += blockDim.x) {
      const int b = b0 + tid, c = b < B ? num[b] : 0;
      const int i = block_inclusive_scan(c > 0, wsum), j = block_inclusive_scan(c, wsum);
      if (c > 0) {
        src[nsrc + i - 1] = (short)b;
        first[nsrc + i - 1] = (short)(nmov + j - c);
        num[b] = nmov + j - c;   // where the next of its rows goes
        if (from[b] != b) sh[2] = 1;
      }
      if (tid == blockDim.x - 1) {
        sh[0] = i;
        sh[1] = j;
      }
      __syncthreads();
      nsrc += sh[0];
      nmov += sh[1];
      __syncthreads();
    }
    for (int b = tid; b < B; b += blockDim.x)
      if (from[b] != b) dst[atomicAdd(&num[from[b]], 1)] = (short)b;
    if (tid == 0) {
      first[nsrc] = (short)nmov;
      sh[0] = nsrc;
      sh[1] = nmov;
    }
    __syncthreads();
  }
  r.nsrc = sh[0];
  r.nmov = sh[1];
  r.chained = sh[2] != 0;
  return r;
}

// Bytes of segment `seg`, from c0 on and at most `bytes`, that a row taken over from source s needs.
__device__ __forceinline__ int row_limit(const RowBuffer& r, int s, int d, int seg, int c0, int bytes) {
  if (!r.counts) return bytes;
  return max(0, min(bytes, max(row_count(r, s, seg), row_count(r, d, seg)) * r.unit - c0));
}

// `bytes` of one source from offset `off` to the rows dst[0..n) (each as far as it needs).
template <typename V>
__device__ __forceinline__ void copy_rows(const RowBuffer& r, long long off, int seg, int c0, int bytes, int s,
                                          const short* dst, int n) {
  constexpr int W = (int)sizeof(V);
  int most = 0;
  for (int i = 0; i < n; ++i) most = max(most, row_limit(r, s, dst[i], seg, c0, bytes));
  const char* from = r.base + s * r.stride + off;
  for (int x = threadIdx.x * W; x < most; x += 4 * kReorderThreads * W) {
    V v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (x + j * kReorderThreads * W < most) v[j] = *reinterpret_cast<const V*>(from + x + j * kReorderThreads * W);
    for (int i = 0; i < n; ++i) {
      const int d = dst[i], lim = row_limit(r, s, d, seg, c0, bytes);
      char* to = r.base + d * r.stride + off;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (x + j * kReorderThreads * W < lim) *reinterpret_cast<V*>(to + x + j * kReorderThreads * W) = v[j];
    }
  }
}

// A column of all sources (C bytes each) into the stage, a warp to a source.
template <typename V>
__device__ __forceinline__ void stage_in(const RowBuffer& r, long long off, int C, int nsrc, const short* src,
                                         const int* lim, char* stage) {
  for (int s = threadIdx.x >> 5; s < nsrc; s += kReorderThreads / 32) {
    const char* from = r.base + src[s] * r.stride + off;
    for (int c = (threadIdx.x & 31) * (int)sizeof(V); c < lim[s]; c += 32 * (int)sizeof(V)) {
      if (sizeof(V) == 16) cp_async16(stage + s * C + c, from + c);
      else *reinterpret_cast<V*>(stage + s * C + c) = *reinterpret_cast<const V*>(from + c);
    }
  }
}
template <typename V>
__device__ __forceinline__ void stage_out(const RowBuffer& r, long long off, int C, int nsrc, const short* src,
                                          const short* first, const short* dst, int seg, int c0, int bytes,
                                          const char* stage) {
  for (int s = threadIdx.x >> 5; s < nsrc; s += kReorderThreads / 32)
    for (int i = first[s]; i < first[s + 1]; ++i) {
      char* to = r.base + dst[i] * r.stride + off;
      const int lim = row_limit(r, src[s], dst[i], seg, c0, bytes);
      for (int c = (threadIdx.x & 31) * (int)sizeof(V); c < lim; c += 32 * (int)sizeof(V))
        *reinterpret_cast<V*>(to + c) = *reinterpret_cast<const V*>(stage + s * C + c);
    }
}

template <typename F>
__device__ __forceinline__ void by_width(int width, F f) {
  switch (width) {
    case 16: f(uint4{}); break;
    case 8: f(uint2{}); break;
    case 4: f(0u); break;
    case 2: f((unsigned short)0); break;
    default: f((unsigned char)0); break;
  }
}

__global__ void __launch_bounds__(kReorderThreads, 4) reorder_kernel(const __grid_constant__ RowArgs a, int stage_bytes) {
  extern __shared__ uint4 smem4[];
  char* stage = reinterpret_cast<char*>(smem4);
  int* num = reinterpret_cast<int*>(stage + stage_bytes);   // [B]
  short* src = reinterpret_cast<short*>(num + a.B);         // [B]
  short* first = src + a.B;                                 // [B + 1]
  short* dst = first + a.B + 1;                             // [B]
  short* from = dst + a.B;                                  // [B]
  pdl_entry();
  const RowLists l = row_lists(a, src, first, dst, from, num);
  if (l.nmov == 0) return;
  const int tid = threadIdx.x;
  // Tiles: (buffer, segment, column, source), or all sources of a column together when they are staged.
  const int C = l.chained ? min(stage_bytes / l.nsrc, kReorderTile) & ~63 : kReorderTile;
  const int split = l.chained ? 1 : l.nsrc;
  // Tiles before each buffer (fewer than 2^31: each moves 64 bytes or more of every source).
  __shared__ int begin[kRowBuffers + 1], cols[kRowBuffers];
  if (tid == 0) begin[0] = 0;
  if (tid < 64) {
    const int c = tid < a.n ? (a.buf[tid].seg_bytes + C - 1) / C : 0;
    int v = tid < a.n ? c * a.buf[tid].segs * split : 0;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, v, off);
      if ((tid & 31) >= off) v += y;
    }
    if (tid < a.n) {
      cols[tid] = c;
      begin[tid + 1] = v;
    }
  }
  __syncthreads();
  if (tid >= 32 && tid < a.n) begin[tid + 1] += begin[32];
  __syncthreads();
  int i = 0;
  for (int id = blockIdx.x; id < begin[a.n]; id += gridDim.x) {
    while (id >= begin[i + 1]) ++i;
    const RowBuffer& r = a.buf[i];
    const int t = id - begin[i], at = t / split, s = t - at * split, seg = at / cols[i], c0 = (at - seg * cols[i]) * C;
    const int bytes = min(C, r.seg_bytes - c0);
    const long long off = (long long)seg * r.seg_stride + c0;
    if (!l.chained) {
      by_width(r.width, [&](auto v) {
        copy_rows<decltype(v)>(r, off, seg, c0, bytes, l.src[s], l.dst + l.first[s], l.first[s + 1] - l.first[s]);
      });
      continue;
    }
    __syncthreads();   // the stage and the limits of the previous tile have been read
    for (int x = tid; x < l.nsrc; x += kReorderThreads) {
      int lim = 0;
      for (int j = l.first[x]; j < l.first[x + 1]; ++j) lim = max(lim, row_limit(r, l.src[x], l.dst[j], seg, c0, bytes));
      num[x] = lim;
    }
    __syncthreads();
    by_width(r.width, [&](auto v) { stage_in<decltype(v)>(r, off, C, l.nsrc, l.src, num, stage); });
    cp_async_commit();
    cp_async_wait<0>();
    __syncthreads();
    by_width(r.width, [&](auto v) {
      stage_out<decltype(v)>(r, off, C, l.nsrc, l.src, l.first, l.dst, seg, c0, bytes, stage);
    });
  }
}

// The counts themselves, once nothing reads them any more: whole rows of the (small) buffers through shared
// memory, 64 bytes of every row per CTA.
__global__ void __launch_bounds__(kReorderThreads) reorder_counts_kernel(const __grid_constant__ RowArgs a) {
  extern __shared__ uint4 smem4[];
  unsigned short* old = reinterpret_cast<unsigned short*>(smem4);   // [B][32]
  pdl_entry();
  const RowBuffer& r = a.buf[blockIdx.y];
  const int lane = threadIdx.x & 31, c = (blockIdx.x * 32 + lane) * 2;
  if (c < r.seg_bytes)
    for (int b = threadIdx.x >> 5; b < a.B; b += kReorderThreads / 32)
      old[b * 32 + lane] = *reinterpret_cast<const unsigned short*>(r.base + b * r.stride + c);
  __syncthreads();
  for (int b = threadIdx.x >> 5; b < a.B; b += kReorderThreads / 32) {
    const int s = source_of(a, b);
    if (s != b && c < r.seg_bytes) *reinterpret_cast<unsigned short*>(r.base + b * r.stride + c) = old[s * 32 + lane];
  }
}

// ---------------------------------------------------------------- host side
static void add_rows(RowArgs* a, void* base, long long stride, int segs, long long seg_stride, long long seg_bytes,
                     const void* counts = nullptr, int count_size = 0, int unit = 0) {
  if (segs < 1 || seg_bytes < 1) return;
  RowBuffer& r = a->buf[a->n++];
  r.base = static_cast<char*>(base);
  r.counts = counts;
  r.stride = stride;
  r.seg_stride = seg_stride;
  r.segs = segs;
  r.seg_bytes = (int)seg_bytes;
  r.unit = unit;
  r.count_size = (short)count_size;
  const unsigned long long all = (unsigned long long)reinterpret_cast<uintptr_t>(base) | (unsigned long long)stride |
                                 (segs > 1 ? (unsigned long long)seg_stride : 0ull) | (unsigned long long)seg_bytes |
                                 (unsigned long long)unit;
  r.width = 16;
  while (all % r.width) r.width /= 2;
}

static size_t reorder_stage(int B) { return std::max<size_t>(kReorderStage, (size_t)B * 64); }

static void set_index(RowArgs& a, int B, const void* index, int wide, int32_t* status) {
  a.B = B;
  a.index = index;
  a.wide = wide;
  a.status = status;
}

static int launch_reorder(RowArgs& a, int B, const void* index, int wide, int32_t* status, cudaStream_t st) {
  if (a.n == 0) return LOGKV_OK;
  set_index(a, B, index, wide, status);
  const size_t stage = reorder_stage(B), smem = stage + (size_t)B * 12 + 16;
  const cudaError_t e = cudaFuncSetAttribute(reorder_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return (int)e;
  // The CTAs loop over the tiles; no more CTAs than a source per row would need.
  long long tiles = 0;
  for (int i = 0; i < a.n; ++i)
    tiles += (long long)(a.buf[i].seg_bytes + kReorderTile - 1) / kReorderTile * a.buf[i].segs * B;
  const int per_sm = (int)std::max<size_t>(1, std::min<size_t>(4, (220 * 1024) / (smem + 1024)));
  launch_pdl(reorder_kernel, dim3((unsigned)std::max(1LL, std::min<long long>(tiles, 148LL * per_sm))),
             kReorderThreads, smem, st, a, (int)stage);
  return launch_status();
}

static int launch_counts(RowArgs& a, int B, const void* index, int wide, int32_t* status, cudaStream_t st) {
  set_index(a, B, index, wide, status);
  int cols = 1;
  for (int i = 0; i < a.n; ++i) cols = std::max(cols, (a.buf[i].seg_bytes + 63) / 64);
  const size_t smem = (size_t)B * 64;
  const cudaError_t e = cudaFuncSetAttribute(reorder_counts_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return (int)e;
  launch_pdl(reorder_counts_kernel, dim3(cols, a.n), kReorderThreads, smem, st, a);
  return launch_status();
}

}  // namespace logkv

using namespace logkv;

extern "C" {

LOGKV_API int logkv_reorder_batch(const logkv_layout_t* layout, const logkv_state_t* state,
                                  const logkv_prefix_t* prefix, int32_t recent_count, int32_t window_from,
                                  const void* index, int32_t index_wide, int32_t* status, void* stream) {
  if (!layout || !state || !index) return LOGKV_E_POINTER;
  const logkv_layout_t& l = *layout;
  if (l.dtype != LOGKV_DTYPE_F32 && l.dtype != LOGKV_DTYPE_BF16) return LOGKV_E_DTYPE;
  if (l.batch < 1 || l.batch > kReorderBatch || l.groups < 1 || l.dim < 1 || l.clusters < 1 || l.levels < 1 ||
      l.slots < 1 || l.exact < 1 || recent_count < 0 || recent_count > l.recent_capacity || window_from < -1 ||
      window_from > recent_count || (prefix && prefix->capacity < 1))
    return LOGKV_E_SHAPE;
  const logkv_state_t& s = *state;
  const void* all[] = {s.level_k,  s.level_v,    s.level_w,   s.level_p_lo,  s.level_p_hi,  s.level_sum_wp, s.level_order,
                       s.pad_mask, s.level_count, s.centroid, s.n_eff,       s.n_total,     s.p_hi_c,       s.level0_phase,
                       s.alive,    s.s_h,        s.recent_k,  s.recent_k_raw, s.recent_v,   s.recent_pos,   s.recent_ends,
                       s.alpha_k_raw, s.alpha_v, s.alpha_pos, s.alpha_valid, s.alpha_span_len, s.alpha_span_closed,
                       s.alpha_nspans, s.alpha_rowcount};
  for (const void* p : all)
    if (!p) return LOGKV_E_POINTER;
  if (prefix && (!prefix->k || !prefix->v || !prefix->mass || !prefix->length)) return LOGKV_E_POINTER;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const long long e = l.dtype == LOGKV_DTYPE_BF16 ? 2 : 4, G = l.groups, D = l.dim, K = l.clusters, P = l.exact;
  const long long cap = l.recent_capacity, KL = K * l.levels, Bs = l.slots, cells = KL * Bs;
  if (Bs * D * e > (1LL << 30) || G * cells * 8 > (1LL << 30) || cap * D * e > (1LL << 30) || P * D * e > (1LL << 30) ||
      (prefix && prefix->capacity * D * e > (1LL << 30)) || G * K * D * 4 > (1LL << 30))
    return LOGKV_E_SHAPE;
  RowArgs a{};
  const long long w0 = window_from < 0 ? 0 : window_from, wn = recent_count - w0;
  // The window's rows [w0, recent_count) of every group.
  for (void* p : {s.recent_k, s.recent_k_raw, s.recent_v})
    add_rows(&a, static_cast<char*>(p) + w0 * D * e, G * cap * D * e, (int)G, cap * D * e, wn * D * e);
  add_rows(&a, s.recent_pos + w0, cap * 8, 1, 0, wn * 8);
  add_rows(&a, s.recent_ends + w0, cap, 1, 0, wn);
  if (window_from >= 0) return launch_reorder(a, l.batch, index, index_wide, status, st);
  auto rows = [&](void* p, long long bytes) { add_rows(&a, p, bytes, 1, 0, bytes); };
  for (void* p : {s.level_k, s.level_v})
    add_rows(&a, p, G * cells * D * e, (int)(G * KL), Bs * D * e, Bs * D * e, s.level_count, 2, (int)(D * e));
  if (prefix) {
    for (void* p : {prefix->k, prefix->v})
      add_rows(&a, p, G * prefix->capacity * D * e, (int)G, prefix->capacity * D * e, prefix->capacity * D * e,
               prefix->length, 4, (int)(D * e));
    add_rows(&a, prefix->mass, G * prefix->capacity * 4, (int)G, prefix->capacity * 4LL, prefix->capacity * 4LL,
             prefix->length, 4, 4);
  }
  for (void* p : {s.alpha_k_raw, s.alpha_v}) rows(p, G * P * D * e);
  // A slot's bookkeeping (37 bytes beside its 2 D e of K and V) moves as whole rows: its short
  // segments are not 16-byte aligned.
  rows(s.level_w, G * cells * 4);
  for (int64_t* p : {s.level_p_lo, s.level_p_hi, s.level_sum_wp, s.level_order}) rows(p, G * cells * 8);
  rows(s.pad_mask, G * cells);
  rows(s.centroid, G * K * D * 4);
  rows(s.n_eff, G * K * 4);
  rows(s.n_total, G * K * 4);
  rows(s.p_hi_c, G * K * 8);
  rows(s.level0_phase, G * K * 4);
  rows(s.alive, G * K);
  rows(s.s_h, G * 4);
  rows(s.alpha_pos, P * 8);
  rows(s.alpha_valid, P);
  rows(s.alpha_span_len, P * 4);
  rows(s.alpha_span_closed, P);
  rows(s.alpha_nspans, 4);
  rows(s.alpha_rowcount, 4);
  const int rc = launch_reorder(a, l.batch, index, index_wide, status, st);
  if (rc) return rc;
  // The counts, once nothing reads them any more.
  RowArgs c{};
  add_rows(&c, s.level_count, G * KL * 2, 1, 0, G * KL * 2);
  if (prefix) add_rows(&c, prefix->length, G * 4, 1, 0, G * 4);
  return launch_counts(c, l.batch, index, index_wide, status, st);
}

LOGKV_API int logkv_reorder_rows(const logkv_rows_t* buffers, int32_t n, int32_t batch, const void* index,
                                 int32_t index_wide, int32_t* status, void* stream) {
  if (!buffers || !index) return LOGKV_E_POINTER;
  if (n < 0 || n > kRowBuffers || batch < 1 || batch > kReorderBatch) return LOGKV_E_SHAPE;
  RowArgs a{};
  for (int i = 0; i < n; ++i) {
    if (!buffers[i].base) return LOGKV_E_POINTER;
    if (buffers[i].row_bytes < 0 || buffers[i].row_bytes > (1LL << 30)) return LOGKV_E_SHAPE;
    add_rows(&a, buffers[i].base, buffers[i].row_bytes, 1, 0, buffers[i].row_bytes);
  }
  return launch_reorder(a, batch, index, index_wide, status, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
