// Batch rows of a cache taken over by the hypotheses that go on (C ABI in include/logkv_b200.h):
// row b of every state buffer becomes the old row index[b], in place.
//
// A buffer's batch row is `segs` segments of bytes; rows that stay are neither read nor written.  A warp
// moves a column of up to 8 KB of a segment at a time by bulk copies, through a ring of shared-memory
// slots: source rows in, every row that takes one over out, four columns on their way in while earlier
// ones go out, so one CTA of four warps keeps 190 KB of an SM in motion and issues next to nothing.  Where
// every source row stays itself (beams that go on keep their places) a column is of one source.  Where a
// source row is itself taken over (swaps, chains, cycles) it is of all sources: they are in shared
// memory before any row is written and no other warp touches the column, so the rows need no order and
// the state no second copy.
//
// Bound by HBM: 4 of 8 rows of a 32K-token cache (369 MB to move) take 75 us, 0.76 of the measured copy
// bandwidth (92 us through registers, bound by instructions); a window's tail of 27 of 64 rows 10.8 us, 0.93.
// Where rows change places columns shrink with the number of sources, and copies with them: 8 rows of which
// half move take 75 us, with one swap among them 112, all in rings of four 237; the tail of 64 rows 12, 31 and
// 272.  (A batch's columns are of one kind, so a single swap costs all rows.)
#include <algorithm>

#include "attn_common.cuh"

namespace logkv {

constexpr int32_t kStatusBadIndex = 1 << 19;
constexpr int kRowBuffers = 60;
constexpr int kReorderWarps = 4;
constexpr int kReorderBatch = LOGKV_REORDER_MAX_BATCH;
constexpr int kReorderSlots = 6, kReorderAhead = 4;   // slots of a warp's ring; columns on their way in
constexpr int kReorderSlot = 8 * 1024;                // bytes of a slot
constexpr int kReorderTileBatch = 32;                 // tiles whose places a warp works out together
constexpr long long kReorderWaitBudget = 4000000000LL;   // clock cycles (about 2 s)
constexpr int32_t kStatusReorderTimeout = 1 << 20;

// Segment i of row b: base + b * stride + i * seg_stride, seg_bytes long.  With counts (of element
// size count_size, [B, segs]) only the first unit * max(count of the source, count of the row) bytes
// (rounded up to whole accesses) move: K and V past a level's count are zero in every row (a flush clears
// what it vacates), and prefix rows past the length are never read.
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

__device__ __forceinline__ void bulk_in(void* dst, const void* src, int bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(
                   tc::smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(tc::smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void bulk_out(void* dst, const void* src, int bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\n" ::"l"(dst), "r"(tc::smem_u32(src)),
               "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void bulk_wait_read() {   // all but the last N groups have read their source
  asm volatile("cp.async.bulk.wait_group.read %0;\n" ::"n"(N) : "memory");
}
__device__ __forceinline__ void bulk_wait() { asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory"); }

// A column of one segment: bytes [0, len) at `base` + row * stride, of the sources [s0, s1).
struct RowTile {
  char* base;
  long long stride;
  int len;          // 0: nothing to move
  short s0, s1;
  short width, pad;
};

// Elements of V between the rows and a slot, a lane to an element (buffers too narrow for bulk copies).
template <typename V>
__device__ __forceinline__ void narrow_copy(const RowTile& t, const RowLists& l, int C, char* slot, int lane) {
  const int per = t.len / (int)sizeof(V);
  for (int s = t.s0; s < t.s1; ++s) {
    const V* from = reinterpret_cast<const V*>(t.base + l.src[s] * t.stride);
    V* to = reinterpret_cast<V*>(slot + (s - t.s0) * C);
    for (int x0 = lane; x0 < per; x0 += 8 * 32) {
      V v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (x0 + 32 * j < per) v[j] = from[x0 + 32 * j];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (x0 + 32 * j < per) to[x0 + 32 * j] = v[j];
    }
  }
  __syncwarp();
  for (int s = t.s0; s < t.s1; ++s)
    for (int i = l.first[s]; i < l.first[s + 1]; ++i)
      for (int x = lane; x < per; x += 32)
        reinterpret_cast<V*>(t.base + l.dst[i] * t.stride)[x] = reinterpret_cast<const V*>(slot + (s - t.s0) * C)[x];
  __syncwarp();
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

__global__ void __launch_bounds__(kReorderWarps * 32, 1) reorder_kernel(const __grid_constant__ RowArgs a) {
  extern __shared__ __align__(128) uint4 smem4[];
  char* ring = reinterpret_cast<char*>(smem4);
  int* num = reinterpret_cast<int*>(ring + kReorderWarps * kReorderSlots * kReorderSlot);   // [B]
  short* src = reinterpret_cast<short*>(num + a.B);                                         // [B]
  short* first = src + a.B;                                                                 // [B + 1]
  short* dst = first + a.B + 1;                                                             // [B]
  short* from = dst + a.B;                                                                  // [B]
  __shared__ uint64_t full[kReorderWarps][kReorderSlots];
  __shared__ RowTile tiles[kReorderWarps][kReorderTileBatch];
  __shared__ int begin[kRowBuffers + 1], cols[kRowBuffers];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid < kReorderWarps * kReorderSlots) tc::mbar_init(&full[0][0] + tid, 1);
  tc::mbar_fence_init();
  pdl_entry();
  const RowLists l = row_lists(a, src, first, dst, from, num);
  if (l.nmov == 0) return;
  // Tiles: (buffer, segment, column, source), or all sources of a column together.
  const int each = l.chained ? l.nsrc : 1, split = l.chained ? 1 : l.nsrc, C = kReorderSlot / each & ~15;
  // Tiles before each buffer (fewer than 2^31: each moves 16 bytes or more of every source).
  if (tid == 0) begin[0] = 0;
  if (tid < 64) {
    const int c = tid < a.n ? (a.buf[tid].seg_bytes + C - 1) / C : 0;
    int v = tid < a.n ? c * a.buf[tid].segs * split : 0;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, v, off);
      if (lane >= off) v += y;
    }
    if (tid < a.n) {
      cols[tid] = c;
      begin[tid + 1] = v;
    }
  }
  __syncthreads();
  if (tid >= 32 && tid < a.n) begin[tid + 1] += begin[32];
  __syncthreads();
  char* slots = ring + warp * kReorderSlots * kReorderSlot;
  RowTile* mine = tiles[warp];
  const int stride = gridDim.x * kReorderWarps, total = begin[a.n];
  int in = 0, out = 0;   // columns asked for and written so far
  bool ok = true;
  // One column: wait for its sources, write the rows that take them over.
  auto finish = [&](const RowTile& t) {
    const int slot = out % kReorderSlots;
    ok = ok && __all_sync(0xffffffffu, tc::mbar_wait(&full[warp][slot], (out / kReorderSlots) & 1, kReorderWaitBudget));
    if (ok)
      for (int s = t.s0; s < t.s1; ++s)
        for (int i = l.first[s] + lane; i < l.first[s + 1]; i += 32)
          bulk_out(t.base + l.dst[i] * t.stride, slots + slot * kReorderSlot + (s - t.s0) * C, t.len);
    bulk_commit();
    ++out;
  };
  for (int id0 = blockIdx.x * kReorderWarps + warp; id0 < total && ok; id0 += stride * kReorderTileBatch) {
    // A lane to a tile: its place, and how far its rows go.
    const int id = id0 + lane * stride;
    RowTile t{};
    if (id < total) {
      int i = 0;
      while (id >= begin[i + 1]) ++i;
      const RowBuffer& r = a.buf[i];
      const int q = id - begin[i], at = q / split, s = q - at * split, seg = at / cols[i], c0 = (at - seg * cols[i]) * C;
      t.s0 = (short)(l.chained ? 0 : s);
      t.s1 = (short)(l.chained ? l.nsrc : s + 1);
      t.len = min(C, r.seg_bytes - c0);
      if (r.counts) {
        int n = 0;
        for (int x = t.s0; x < t.s1; ++x) {
          n = max(n, row_count(r, l.src[x], seg));
          for (int j = l.first[x]; j < l.first[x + 1]; ++j) n = max(n, row_count(r, l.dst[j], seg));
        }
        t.len = max(0, min(t.len, (n * r.unit + r.width - 1) / r.width * r.width - c0));
      }
      t.base = r.base + (long long)seg * r.seg_stride + c0;
      t.stride = r.stride;
      t.width = r.width;
    }
    mine[lane] = t;
    __syncwarp();
    const unsigned bulk = __ballot_sync(0xffffffffu, t.len > 0 && t.width == 16);
    unsigned narrow = __ballot_sync(0xffffffffu, t.len > 0 && t.width < 16);
    unsigned ask = bulk, done = bulk;
    while (done && ok) {
      if (ask && in - out < kReorderAhead) {
        const RowTile& n = mine[__ffs(ask) - 1];
        ask &= ask - 1;
        const int slot = in % kReorderSlots;
        // The column that had the slot before was written kReorderSlots - kReorderAhead columns ago or more.
        bulk_wait_read<kReorderSlots - kReorderAhead - 1>();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive_expect_tx(&full[warp][slot], n.len * (n.s1 - n.s0));
        __syncwarp();
        for (int s = n.s0 + lane; s < n.s1; s += 32)
          bulk_in(slots + slot * kReorderSlot + (s - n.s0) * C, n.base + l.src[s] * n.stride, n.len, &full[warp][slot]);
        ++in;
      } else {
        finish(mine[__ffs(done) - 1]);
        done &= done - 1;
      }
    }
    if (narrow && ok) {
      bulk_wait_read<0>();   // the ring is idle: the first slot serves
      __syncwarp();
      for (; narrow; narrow &= narrow - 1) {
        const RowTile& n = mine[__ffs(narrow) - 1];
        by_width(n.width, [&](auto v) { narrow_copy<decltype(v)>(n, l, C, slots, lane); });
      }
      tc::fence_proxy_async();   // before a bulk copy writes the slot again
    }
    __syncwarp();
  }
  bulk_wait();
  if (!ok) {   // (copies that are late may still land in the ring)
    for (; out < in; ++out) tc::mbar_wait(&full[warp][out % kReorderSlots], (out / kReorderSlots) & 1, kReorderWaitBudget);
    if (lane == 0) set_status(a.status, kStatusReorderTimeout);
  }
}

// The counts themselves, once nothing reads them any more: whole rows of the (small) buffers through shared
// memory, 64 bytes of every row per CTA.
__global__ void __launch_bounds__(256) reorder_counts_kernel(const __grid_constant__ RowArgs a) {
  extern __shared__ uint4 smem4[];
  unsigned short* old = reinterpret_cast<unsigned short*>(smem4);   // [B][32]
  pdl_entry();
  const RowBuffer& r = a.buf[blockIdx.y];
  const int lane = threadIdx.x & 31, c = (blockIdx.x * 32 + lane) * 2;
  if (c < r.seg_bytes)
    for (int b = threadIdx.x >> 5; b < a.B; b += 8)
      old[b * 32 + lane] = *reinterpret_cast<const unsigned short*>(r.base + b * r.stride + c);
  __syncthreads();
  for (int b = threadIdx.x >> 5; b < a.B; b += 8) {
    const int s = source_of(a, b);
    if (s != b && c < r.seg_bytes) *reinterpret_cast<unsigned short*>(r.base + b * r.stride + c) = old[s * 32 + lane];
  }
}

// ---------------------------------------------------------------- host side
static void add_rows(RowArgs* a, void* base, long long stride, int segs, long long seg_stride, long long seg_bytes,
                     const void* counts = nullptr, int count_size = 0, int unit = 0) {
  if (segs < 1 || seg_bytes < 1) return;
  unsigned long long all = (unsigned long long)reinterpret_cast<uintptr_t>(base) | (unsigned long long)stride |
                           (segs > 1 ? (unsigned long long)seg_stride : 0ull);
  if (!counts && all % 16 == 0 && seg_bytes > 16 && seg_bytes % 16) {   // the odd end apart
    const long long main = seg_bytes & ~15LL;
    add_rows(a, base, stride, segs, seg_stride, main);
    add_rows(a, static_cast<char*>(base) + main, stride, segs, seg_stride, seg_bytes - main);
    return;
  }
  RowBuffer& r = a->buf[a->n++];
  r.base = static_cast<char*>(base);
  r.counts = counts;
  r.stride = stride;
  r.seg_stride = seg_stride;
  r.segs = segs;
  r.seg_bytes = (int)seg_bytes;
  r.unit = unit;
  r.count_size = (short)count_size;
  all |= (unsigned long long)seg_bytes;
  r.width = 16;
  while (all % r.width) r.width /= 2;
}

static void set_index(RowArgs& a, int B, const void* index, int wide, int32_t* status) {
  a.B = B;
  a.index = index;
  a.wide = wide;
  a.status = status;
}

static size_t reorder_smem(int B) {
  return (size_t)kReorderWarps * kReorderSlots * kReorderSlot + (size_t)B * 12 + 16;
}

static int launch_reorder(RowArgs& a, int B, const void* index, int wide, int32_t* status, cudaStream_t st) {
  if (a.n == 0) return LOGKV_OK;
  set_index(a, B, index, wide, status);
  const size_t smem = reorder_smem(B);
  if (const int e = smem_limit_once<reorder_kernel>(reorder_smem(kReorderBatch))) return e;
  // One CTA per SM; no more warps than a source per row would have tiles.
  long long tiles = 0;
  for (int i = 0; i < a.n; ++i)
    tiles += (long long)(a.buf[i].seg_bytes + kReorderSlot - 1) / kReorderSlot * a.buf[i].segs * B;
  const unsigned grid = (unsigned)std::max(1LL, std::min<long long>((tiles + kReorderWarps - 1) / kReorderWarps, 148LL));
  launch_pdl(reorder_kernel, dim3(grid), kReorderWarps * 32, smem, st, a);
  return launch_status();
}

static int launch_counts(RowArgs& a, int B, const void* index, int wide, int32_t* status, cudaStream_t st) {
  set_index(a, B, index, wide, status);
  int cols = 1;
  for (int i = 0; i < a.n; ++i) cols = std::max(cols, (a.buf[i].seg_bytes + 63) / 64);
  const size_t smem = (size_t)B * 64;
  static_assert(kReorderBatch * 64 <= 48 * 1024, "within the default limit");
  launch_pdl(reorder_counts_kernel, dim3(cols, a.n), 256, smem, st, a);
  return launch_status();
}

}  // namespace logkv

using namespace logkv;

extern "C" {

LOGKV_API int logkv_reorder_batch(const logkv_layout_t* layout, const logkv_state_t* state,
                                  const logkv_prefix_t* prefix, int32_t recent_count, int32_t window_from,
                                  const void* index, int32_t index_wide, int32_t* status, void* stream) {
  if (!layout || !state || !index || (reinterpret_cast<uintptr_t>(index) & (index_wide ? 7 : 3))) return LOGKV_E_POINTER;
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
  if (!buffers || !index || (reinterpret_cast<uintptr_t>(index) & (index_wide ? 7 : 3))) return LOGKV_E_POINTER;
  if (n < 0 || n > 30 || batch < 1 || batch > kReorderBatch) return LOGKV_E_SHAPE;
  RowArgs a{};
  for (int i = 0; i < n; ++i) {
    if (!buffers[i].base) return LOGKV_E_POINTER;
    if (buffers[i].row_bytes < 0 || buffers[i].row_bytes > (1LL << 30)) return LOGKV_E_SHAPE;
    add_rows(&a, buffers[i].base, buffers[i].row_bytes, 1, 0, buffers[i].row_bytes);
  }
  return launch_reorder(a, batch, index, index_wide, status, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
