// Batch rows of a cache taken over by the hypotheses that go on (C ABI in include/logkv_b200.h):
// row b of every state buffer becomes the old row index[b], in place.
//
// A buffer's batch row is `segs` segments of bytes.  A CTA takes one column (up to C bytes of one
// segment) of every row that is a source into shared memory, waits, and writes it to the rows that
// take it over; no other CTA touches that column, so chains, swaps and cycles of rows need no order
// and no second copy of the state.  Rows that stay are neither read nor written.
#include <algorithm>

#include "common.cuh"
#include "../../include/logkv_attention.h"

namespace logkv {

constexpr int32_t kStatusBadIndex = 1 << 19;
constexpr int kRowBuffers = 40;
constexpr int kReorderThreads = 256;
constexpr int kReorderBatch = 2048;
constexpr int kReorderStage = 32 * 1024;   // staged bytes per CTA (more above 512 source rows)

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

template <typename V>
__device__ __forceinline__ void stage_in(const RowBuffer& r, long long off, int C, int nsrc, const short* ssrc,
                                         const int* lim, char* stage) {
  const int per = C / (int)sizeof(V);
  for (int x = threadIdx.x; x < nsrc * per; x += blockDim.x) {
    const int s = x / per, c = (x - s * per) * (int)sizeof(V);
    if (c < lim[s]) *reinterpret_cast<V*>(stage + s * C + c) = *reinterpret_cast<const V*>(r.base + ssrc[s] * r.stride + off + c);
  }
}
template <typename V>
__device__ __forceinline__ void stage_out(const RowBuffer& r, long long off, int C, int nmov, const short* mdst,
                                          const short* mslot, const int* mlim, const char* stage) {
  const int per = C / (int)sizeof(V);
  for (int x = threadIdx.x; x < nmov * per; x += blockDim.x) {
    const int m = x / per, c = (x - m * per) * (int)sizeof(V);
    if (c < mlim[m]) *reinterpret_cast<V*>(r.base + mdst[m] * r.stride + off + c) = *reinterpret_cast<const V*>(stage + mslot[m] * C + c);
  }
}

__global__ void __launch_bounds__(kReorderThreads) reorder_kernel(const __grid_constant__ RowArgs a, int stage_bytes) {
  extern __shared__ uint4 smem4[];
  __shared__ int wsum[32];
  __shared__ int sh_n[2];
  char* stage = reinterpret_cast<char*>(smem4);
  int* mlim = reinterpret_cast<int*>(stage + stage_bytes);   // [B] bytes of the column each taken-over row needs
  int* slim = mlim + a.B;                                    // [B] and each source
  short* mdst = reinterpret_cast<short*>(slim + a.B);        // [B] rows taken over
  short* mslot = mdst + a.B;                                 // [B] their source's place in the stage
  short* ssrc = mslot + a.B;                                 // [B] source rows
  short* slot = ssrc + a.B;                                  // [B] place of a source row, -1: none
  const int tid = threadIdx.x, B = a.B;
  pdl_entry();
  auto source = [&](int b) {
    const long long v = a.wide ? static_cast<const long long*>(a.index)[b] : (long long)static_cast<const int32_t*>(a.index)[b];
    if (v >= 0 && v < B) return (int)v;
    if (blockIdx.x == 0) set_status(a.status, kStatusBadIndex);
    return b;
  };
  for (int b = tid; b < B; b += blockDim.x) slot[b] = -1;
  __syncthreads();
  for (int b = tid; b < B; b += blockDim.x) {
    const int s = source(b);
    if (s != b) slot[s] = 0;
  }
  __syncthreads();
  int nsrc = 0, nmov = 0;
  for (int b0 = 0; b0 < B; b0 += blockDim.x) {
    const int b = b0 + tid;
    const bool is = b < B && slot[b] == 0, mv = b < B && source(b) != b;
    const int i = block_inclusive_scan(is, wsum), j = block_inclusive_scan(mv, wsum);
    if (is) {
      ssrc[nsrc + i - 1] = (short)b;
      slot[b] = (short)(nsrc + i - 1);
    }
    if (mv) mdst[nmov + j - 1] = (short)b;
    if (tid == blockDim.x - 1) {
      sh_n[0] = i;
      sh_n[1] = j;
    }
    __syncthreads();
    nsrc += sh_n[0];
    nmov += sh_n[1];
    __syncthreads();
  }
  if (nmov == 0) return;
  for (int m = tid; m < nmov; m += blockDim.x) mslot[m] = slot[source(mdst[m])];
  const int C = min(stage_bytes / nsrc, 16 * 1024) & ~63;
  int i = 0;
  long long first = 0;   // first tile of buffer i
  for (long long id = blockIdx.x;; id += gridDim.x) {
    int cols = 0;
    while (i < a.n) {
      cols = (a.buf[i].seg_bytes + C - 1) / C;
      const long long tiles = (long long)cols * a.buf[i].segs;
      if (id - first < tiles) break;
      first += tiles;
      ++i;
    }
    if (i >= a.n) return;
    const RowBuffer& r = a.buf[i];
    const int seg = (int)((id - first) / cols), c0 = (int)((id - first) % cols) * C;
    const int bytes = min(C, r.seg_bytes - c0);
    __syncthreads();   // the stage and the limits of the previous tile have been read
    for (int s = tid; s < nsrc; s += blockDim.x) slim[s] = r.counts ? 0 : bytes;
    __syncthreads();
    for (int m = tid; m < nmov; m += blockDim.x) {
      int lim = bytes;
      if (r.counts) {
        const int n = max(row_count(r, mdst[m], seg), row_count(r, ssrc[mslot[m]], seg));
        lim = max(0, min(bytes, n * r.unit - c0));
        atomicMax(&slim[mslot[m]], lim);
      }
      mlim[m] = lim;
    }
    __syncthreads();
    const long long off = (long long)seg * r.seg_stride + c0;
    switch (r.width) {
      case 16: stage_in<uint4>(r, off, C, nsrc, ssrc, slim, stage); break;
      case 8: stage_in<uint2>(r, off, C, nsrc, ssrc, slim, stage); break;
      case 4: stage_in<unsigned>(r, off, C, nsrc, ssrc, slim, stage); break;
      case 2: stage_in<unsigned short>(r, off, C, nsrc, ssrc, slim, stage); break;
      default: stage_in<unsigned char>(r, off, C, nsrc, ssrc, slim, stage); break;
    }
    __syncthreads();
    switch (r.width) {
      case 16: stage_out<uint4>(r, off, C, nmov, mdst, mslot, mlim, stage); break;
      case 8: stage_out<uint2>(r, off, C, nmov, mdst, mslot, mlim, stage); break;
      case 4: stage_out<unsigned>(r, off, C, nmov, mdst, mslot, mlim, stage); break;
      case 2: stage_out<unsigned short>(r, off, C, nmov, mdst, mslot, mlim, stage); break;
      default: stage_out<unsigned char>(r, off, C, nmov, mdst, mslot, mlim, stage); break;
    }
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

static int launch_reorder(RowArgs& a, int B, const void* index, int wide, int32_t* status, cudaStream_t st) {
  if (a.n == 0) return LOGKV_OK;
  a.B = B;
  a.index = index;
  a.wide = wide;
  a.status = status;
  const size_t stage = reorder_stage(B), smem = stage + (size_t)B * 16;
  const cudaError_t e = cudaFuncSetAttribute(reorder_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return (int)e;
  // The CTAs loop over columns of about stage / B bytes or more; no more CTAs than columns.
  long long tiles = 0;
  const long long c = std::max<long long>(64, (long long)(stage / B) & ~63LL);
  for (int i = 0; i < a.n; ++i) tiles += (a.buf[i].seg_bytes + c - 1) / c * a.buf[i].segs;
  const int per_sm = (int)std::max<size_t>(1, (220 * 1024) / (smem + 1024));
  launch_pdl(reorder_kernel, dim3((unsigned)std::max(1LL, std::min<long long>(tiles, 148LL * std::min(per_sm, 6)))),
             kReorderThreads, smem, st, a, (int)stage);
  const cudaError_t r = cudaGetLastError();
  return r == cudaSuccess ? LOGKV_OK : (int)r;
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
  return launch_reorder(c, l.batch, index, index_wide, status, st);
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
