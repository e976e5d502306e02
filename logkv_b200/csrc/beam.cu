// Beam search's selection over beams and vocabulary (C ABI in include/logkv_beam.h).
//
//   B1 beam_slice_kernel  one CTA per slice of a beam's vocabulary: one read of the logits gives the
//                          slice's sum of exponentials and its k best logits;
//   B2 beam_merge_kernel  one CTA per request: every beam's log-sum-exp from its slices, then the k
//                          best of all slices' lists by score.
//
// Both find a threshold first: the threads are put into at least 2 k groups, and the k-th largest of
// the groups' maxima has at least k elements at or above it and, unless the values are very uneven, not
// many more; those are gathered and ranked by counting.  When too many are at or above it (ties), the
// k-th largest key is found bit by bit instead.  Keys are (value, lower index first), so the choice is
// unique whatever the order of the gathering.
#include <algorithm>

#include "common.cuh"
#include "tcgen05.cuh"
#include "../../include/logkv_beam.h"

namespace logkv {

constexpr int kBeamThreads = 256;
constexpr int kBeamCand = 1024;    // gathered candidates at most
constexpr int kBeamVecs = 4;       // 16-byte vectors per thread and chunk

struct BeamGeo {
  const void* logits;
  const float* scores;
  float* out_scores;
  long long* out_rows;
  long long* out_tokens;
  long long n_stride, w_stride;
  int W, V, k, S, keep;
  int chunks;     // chunks (kBeamThreads x kBeamVecs vectors) of a beam's vocabulary, divided among S slices
  // Scratch: per (request, beam, slice) the sum of 2^((x - top) e') and top; per request [k][W * S] lists.
  double* sum;
  float* top;
  float* val;
  int* idx;
};

// Monotone map of a float (double) to an unsigned integer; 0 is below every number's.
__device__ __forceinline__ unsigned order32(float x) {
  const unsigned u = __float_as_uint(x + 0.f);   // -0 as +0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned long long order64(double x) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(x + 0.0);
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

template <typename T>
__device__ __forceinline__ T warp_max(T v) {
#pragma unroll
  for (int off = 16; off; off >>= 1) {
    const T o = __shfl_xor_sync(0xffffffffu, v, off);
    v = o > v ? o : v;
  }
  return v;
}

// Sum of one int per thread over the block, to every thread.
__device__ __forceinline__ int block_sum(int v, int* sh) {
#pragma unroll
  for (int off = 16; off; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  int t = 0;
#pragma unroll
  for (int w = 0; w < kBeamThreads / 32; ++w) t += sh[w];
  __syncthreads();
  return t;
}

// The k-th largest of the groups' maxima (0 when fewer groups hold anything); 64 to 256 groups, at least
// 2 k.  `gm`: one entry per thread.
template <typename K>
__device__ __forceinline__ K group_threshold(K mine, int k, K* gm, K* sh) {
  const int gs = k <= 32 ? 4 : k <= 64 ? 2 : 1, ng = kBeamThreads / gs, tid = threadIdx.x;
  for (int off = 1; off < gs; off <<= 1) {
    const K o = __shfl_xor_sync(0xffffffffu, mine, off);
    mine = o > mine ? o : mine;
  }
  if (tid % gs == 0) gm[tid / gs] = mine;
  if (tid == 0) *sh = 0;
  __syncthreads();
  if (tid < ng) {
    const K me = gm[tid];
    int above = 0;
#pragma unroll 8
    for (int g = 0; g < ng; ++g) above += gm[g] > me || (gm[g] == me && g < tid);
    if (above == k - 1) *sh = me;
  }
  __syncthreads();
  return *sh;
}

// ---------------------------------------------------------------- B1
// The logits of one 32-bit word.
template <typename T>
struct BeamWord;
template <>
struct BeamWord<float> {
  static constexpr int N = 1;
  static constexpr unsigned kNone = 0xff800000u;   // -inf
  __device__ __forceinline__ static float get(unsigned w, int) { return __uint_as_float(w); }
  __device__ __forceinline__ static unsigned mask(unsigned w, int) { return kNone; }
  __device__ __forceinline__ static unsigned max(unsigned a, unsigned b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }
  __device__ __forceinline__ static float top(unsigned w) { return __uint_as_float(w); }
};
template <>
struct BeamWord<__nv_bfloat16> {
  static constexpr int N = 2;
  static constexpr unsigned kNone = 0xff80ff80u;
  __device__ __forceinline__ static float get(unsigned w, int e) {
    return __uint_as_float(e ? w & 0xffff0000u : w << 16);
  }
  __device__ __forceinline__ static unsigned mask(unsigned w, int e) {
    return e ? (w & 0xffffu) | 0xff800000u : (w & 0xffff0000u) | 0xff80u;
  }
  __device__ __forceinline__ static unsigned max(unsigned a, unsigned b) {   // NaN gives way
    const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const unsigned*>(&m);
  }
  __device__ __forceinline__ static float top(unsigned w) { return fmaxf(get(w, 0), get(w, 1)); }
};

// Keys of candidates: value, then the lower vocabulary index.
__device__ __forceinline__ unsigned long long beam_key(float x, int v) {
  return (unsigned long long)order32(x) << 32 | (0xffffffffu - (unsigned)v);
}
__device__ __forceinline__ float key_value(unsigned long long key) {
  const unsigned o = (unsigned)(key >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// log2 e as float32.  Sums are of 2^((x - m) e') with e' this constant: log2 of the sum over e' is off from
// its true value by the constant's relative error, 1.3e-8, times the distribution's entropy in nats
// (below 2e-7), the same way for every beam.
constexpr float kLog2e = 1.44269502f;

// A CTA walks its slice in chunks, the next chunk's loads in flight.  Every thread keeps the running
// maximum and sum of its own terms.  Candidates above the running threshold go to a buffer; a buffer
// that fills up is cut to its k best, which raises the threshold.  The first chunk's threshold comes from
// the groups' maxima.  Later elements equal to the threshold are not needed: k elements at or above it
// have lower indices.
template <typename T>
__global__ void __launch_bounds__(kBeamThreads, 4) beam_slice_kernel(BeamGeo a) {
  using U64 = unsigned long long;
  using Word = BeamWord<T>;
  constexpr int WN = Word::N, VN = 4 * WN, NV = kBeamVecs, NW = 4 * NV, CH = kBeamThreads * NV;
  __shared__ unsigned gm[kBeamThreads];
  __shared__ unsigned sh_t;
  __shared__ U64 cand[kBeamCand];
  __shared__ float wmax[kBeamThreads / 32];
  __shared__ double wsum[kBeamThreads / 32];
  __shared__ int isum[kBeamThreads / 32];
  __shared__ int sh_n;
  __shared__ float sh_cut;
  __shared__ unsigned xs[NW * kBeamThreads];
  pdl_entry();
  const int tid = threadIdx.x, slice = blockIdx.x, w = blockIdx.y % a.W, n = blockIdx.y / a.W, k = a.k;
  // The row from the 16-byte boundary at or below its start: element e of it is logit e - lead.
  const T* row = static_cast<const T*>(a.logits) + n * a.n_stride + w * a.w_stride;
  const int lead = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  const uint4* vec = reinterpret_cast<const uint4*>(row - lead);
  const int nvec = (a.V + lead + VN - 1) / VN;
  const int c0 = (int)((long long)a.chunks * slice / a.S), c1 = (int)((long long)a.chunks * (slice + 1) / a.S);
  // Cut the buffer's m entries (m >= 1) to the k best, sorted; the k-th's value is the new threshold.
  auto cut = [&](int m) {
    U64 mine[kBeamCand / kBeamThreads];
    int rank[kBeamCand / kBeamThreads];
#pragma unroll
    for (int i = 0; i < kBeamCand / kBeamThreads; ++i) {
      const int at = tid + i * kBeamThreads;
      mine[i] = at < m ? cand[at] : 0ull;
      rank[i] = at < m ? 0 : k;
      if (at < m) {
#pragma unroll 8
        for (int j = 0; j < m; ++j) rank[i] += cand[j] > mine[i];
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBeamCand / kBeamThreads; ++i)
      if (rank[i] < k) {
        cand[rank[i]] = mine[i];
        if (rank[i] == k - 1) sh_cut = key_value(mine[i]);
      }
    if (tid == 0) sh_n = min(m, k);
    __syncthreads();
  };
  unsigned next[NW], x[NW];
  auto fetch = [&](int c) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = c * CH + i * kBeamThreads + tid;
      uint4 v = make_uint4(Word::kNone, Word::kNone, Word::kNone, Word::kNone);
      if (j < nvec) v = __ldcs(vec + j);
      next[4 * i] = v.x, next[4 * i + 1] = v.y, next[4 * i + 2] = v.z, next[4 * i + 3] = v.w;
    }
  };
  // Vocabulary index of element e of the thread's word i in chunk c.
  auto index = [&](int c, int i, int e) { return (c * CH + i / 4 * kBeamThreads + tid) * VN + i % 4 * WN + e - lead; };
  if (tid == 0) {
    sh_n = 0;
    sh_cut = -INFINITY;
  }
  const int full = max(4 * k, 128);   // entries that call for a cut
  float cutoff = -INFINITY, m = -INFINITY, s = 0.f;
  fetch(c0);
  for (int c = c0; c < c1; ++c) {
#pragma unroll
    for (int i = 0; i < NW; ++i) x[i] = next[i];
    if (c == 0 || (c + 1) * CH >= nvec) {   // the row's first and last vectors may hold a neighbour's logits
#pragma unroll
      for (int i = 0; i < NW; ++i)
#pragma unroll
        for (int e = 0; e < WN; ++e) {
          const int v = index(c, i, e);
          if (v < 0 || v >= a.V) x[i] = Word::mask(x[i], e);
        }
    }
    if (c + 1 < c1) fetch(c + 1);
    unsigned mx = x[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) mx = Word::max(mx, x[i]);
    const float mt = Word::top(mx);
    if (mt > m) {
      s = m == -INFINITY ? s : s * tc::ex2((m - mt) * kLog2e);   // s without a finite maximum: 0 or NaN
      m = mt;
    }
    const float ref = m == -INFINITY ? 0.f : m;
    const uint64_t e2 = tc::f2pack(kLog2e, kLog2e), m2 = tc::f2pack(-ref, -ref);
    uint64_t s2 = tc::f2pack(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NW; i += 2 / WN) {
      const float x0 = Word::get(x[i], 0), x1 = WN == 2 ? Word::get(x[i], 1) : Word::get(x[(i + 1) % NW], 0);
      float y0, y1;
      tc::f2unpack(tc::fmul2(tc::fadd2(tc::f2pack(x0, x1), m2), e2), y0, y1);
      s2 = tc::fadd2(s2, tc::f2pack(tc::ex2(y0), tc::ex2(y1)));
    }
    float s0, s1;
    tc::f2unpack(s2, s0, s1);
    s += s0 + s1;
    // Candidates of this chunk: above the threshold, in the first chunk at or above the groups'.
    bool first = c == c0;
    if (first) {
      const unsigned none = order32(-INFINITY);
      const unsigned t = max(group_threshold<unsigned>(order32(mt), k, gm, &sh_t), none);
      cutoff = t == none ? -INFINITY : __uint_as_float(t & 0x80000000u ? t & 0x7fffffffu : ~t);
      first = t != none;
    }
    int last = -1;
    if (first ? mt >= cutoff : mt > cutoff) {
#pragma unroll
      for (int i = 0; i < NW; ++i)
#pragma unroll
        for (int e = 0; e < WN; ++e) {
          const float v = Word::get(x[i], e);
          if (first ? v >= cutoff : v > cutoff) {
            last = atomicAdd(&sh_n, 1);
            if (last < kBeamCand) cand[last] = beam_key(v, index(c, i, e));
          }
        }
    }
    if (!__syncthreads_or(last >= full)) continue;
    const int got = sh_n;
    if (got <= kBeamCand) {
      cut(got);
    } else {
      // More than the buffer holds: the k-th largest key of the buffer's earlier entries and this chunk,
      // bit by bit.
      const int begin = c * CH * VN - lead;   // earlier entries have lower indices
      U64 old[kBeamCand / kBeamThreads];
#pragma unroll
      for (int i = 0; i < kBeamCand / kBeamThreads; ++i) {
        old[i] = cand[tid + i * kBeamThreads];
        if ((int)(0xffffffffu - (unsigned)old[i]) >= begin) old[i] = 0ull;
      }
      // (From shared memory: unrolled over registers, the keys would be kept over the 64 rounds.)
#pragma unroll
      for (int i = 0; i < NW; ++i) xs[i * kBeamThreads + tid] = x[i];
      auto key = [&](int q) {
        const int i = q / WN, e = q % WN;
        const float v = Word::get(xs[i * kBeamThreads + tid], e);
        return v > -INFINITY ? beam_key(v, index(c, i, e)) : 0ull;
      };
      U64 kt = 0;
      for (int bit = 63; bit >= 0; --bit) {
        const U64 test = kt | 1ull << bit;
        int cnt = 0;
#pragma unroll 1
        for (int q = 0; q < NW * WN; ++q) cnt += key(q) >= test;
#pragma unroll
        for (int i = 0; i < kBeamCand / kBeamThreads; ++i) cnt += old[i] >= test;
        if (block_sum(cnt, isum) >= k) kt = test;
      }
      if (tid == 0) sh_n = 0;
      __syncthreads();
#pragma unroll 1
      for (int q = 0; q < NW * WN; ++q)
        if (key(q) >= kt) cand[atomicAdd(&sh_n, 1)] = key(q);
#pragma unroll
      for (int i = 0; i < kBeamCand / kBeamThreads; ++i)
        if (old[i] >= kt) cand[atomicAdd(&sh_n, 1)] = old[i];
      __syncthreads();
      cut(k);
    }
    cutoff = sh_cut;
  }
  __syncthreads();
  const int nc = sh_n;
  if (nc) cut(nc);   // sorted
  const float mw = warp_max(m);
  if ((tid & 31) == 0) wmax[tid >> 5] = mw;
  __syncthreads();
  float t = wmax[0];
#pragma unroll
  for (int i = 1; i < kBeamThreads / 32; ++i) t = fmaxf(t, wmax[i]);
  double sd = m == -INFINITY ? (double)s : (double)s * exp2f((m - t) * kLog2e);   // s is 0 or NaN without a maximum
#pragma unroll
  for (int off = 16; off; off >>= 1) sd += __shfl_xor_sync(0xffffffffu, sd, off);
  if ((tid & 31) == 0) wsum[tid >> 5] = sd;
  __syncthreads();
  const size_t at = (size_t)blockIdx.y * a.S + slice;
  if (tid == 0) {
    double total = 0.0;
    for (int i = 0; i < kBeamThreads / 32; ++i) total += wsum[i];
    a.sum[at] = total;
    a.top[at] = t;
  }
  const int L = a.W * a.S;
  float* val = a.val + (size_t)n * k * L + w * a.S + slice;
  int* idx = a.idx + (size_t)n * k * L + w * a.S + slice;
  for (int i = tid; i < k; i += kBeamThreads) {
    val[(size_t)i * L] = i < nc ? key_value(cand[i]) : 0.f;
    idx[(size_t)i * L] = i < nc ? (int)(0xffffffffu - (unsigned)cand[i]) : -1;
  }
}

// ---------------------------------------------------------------- B2
__global__ void __launch_bounds__(kBeamThreads) beam_merge_kernel(BeamGeo a) {
  using U64 = unsigned long long;
  __shared__ U64 gm[kBeamThreads];
  __shared__ U64 sh_t;
  __shared__ U64 cand[kBeamCand];
  __shared__ int cidx[kBeamCand];
  __shared__ double lse[LOGKV_BEAM_MAX_WIDTH];
  __shared__ int isum[kBeamThreads / 32];
  __shared__ int sh_n;
  __shared__ U64 best[LOGKV_BEAM_MAX_K];
  __shared__ int bflat[LOGKV_BEAM_MAX_K];
  __shared__ short place[LOGKV_BEAM_MAX_K];
  pdl_entry();
  const int tid = threadIdx.x, lane = tid & 31, n = blockIdx.x, W = a.W, S = a.S, k = a.k, L = W * S;
  // log sum exp of each beam in float64; NaN for a beam that offers nothing.
  for (int w = tid >> 5; w < W; w += kBeamThreads / 32) {
    const size_t at = (size_t)(n * W + w) * S;
    float m = -INFINITY;
    for (int i = lane; i < S; i += 32) m = fmaxf(m, a.sum[at + i] > 0.0 ? a.top[at + i] : -INFINITY);
    m = warp_max(m);
    double s = 0.0;
    for (int i = lane; i < S; i += 32) {
      const double si = a.sum[at + i];
      if (si != 0.0) s += si * exp2(((double)a.top[at + i] - (double)m) * kLog2e);   // a NaN stays
    }
#pragma unroll
    for (int off = 16; off; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    if (lane == 0) {
      const float r = a.scores[n * W + w];
      const double z = (double)m + log2(s) / (double)kLog2e;
      lse[w] = isfinite(r) && isfinite(z) ? z : nan("");
    }
  }
  if (tid == 0) sh_n = 0;
  __syncthreads();
  const float* val = a.val + (size_t)n * k * L;
  const int* idx = a.idx + (size_t)n * k * L;
  // Candidate i = place * L + list.  Score key, 0 for none.
  auto key = [&](int i, int& flat) -> U64 {
    const int v = idx[i], w = i % L / S;
    flat = w * a.V + v;
    if (v < 0 || isnan(lse[w])) return 0ull;
    return order64((double)a.scores[n * W + w] + ((double)val[i] - lse[w]));
  };
  const int all = k * L;
  U64 mine = 0;
  int flat;
  for (int i = tid; i < all; i += kBeamThreads) {
    const U64 q = key(i, flat);
    mine = q > mine ? q : mine;
  }
  U64 t = group_threshold<U64>(mine, k, gm, &sh_t);
  t = t ? t : 1;
  int cnt = 0;
  for (int i = tid; i < all; i += kBeamThreads) cnt += key(i, flat) >= t;
  int total = block_sum(cnt, isum);
  int tf = 0x7fffffff;   // flat indices taken at the threshold itself
  if (total > kBeamCand) {
    t = 0;
    for (int bit = 63; bit >= 0; --bit) {
      const U64 test = t | 1ull << bit;
      cnt = 0;
      for (int i = tid; i < all; i += kBeamThreads) cnt += key(i, flat) >= test;
      if (block_sum(cnt, isum) >= k) t = test;
    }
    t = t ? t : 1;
    cnt = 0;
    for (int i = tid; i < all; i += kBeamThreads) cnt += key(i, flat) > t;
    const int need = k - block_sum(cnt, isum);
    int low = 0;   // the `need` lowest flat indices among the ties: flat <= tf
    for (int bit = 30; bit >= 0; --bit) {
      const int test = low | 1 << bit;
      cnt = 0;
      for (int i = tid; i < all; i += kBeamThreads) cnt += key(i, flat) == t && flat < test;
      if (block_sum(cnt, isum) < need) low = test;
    }
    tf = low;
  }
  for (int i = tid; i < all; i += kBeamThreads) {
    const U64 q = key(i, flat);
    if (q > t || (q == t && flat <= tf)) {
      const int at = atomicAdd(&sh_n, 1);
      cand[at] = q;
      cidx[at] = flat;
    }
  }
  __syncthreads();
  const int nc = sh_n, found = min(nc, k);
  for (int i = tid; i < nc; i += kBeamThreads) {
    const U64 me = cand[i];
    const int mf = cidx[i];
    int above = 0;
    for (int j = 0; j < nc; ++j) above += cand[j] > me || (cand[j] == me && cidx[j] < mf);
    if (above < k) {
      best[above] = me;
      bflat[above] = mf;
    }
  }
  __syncthreads();
  if (!a.keep) {
    for (int i = tid; i < k; i += kBeamThreads) place[i] = (short)i;
  } else if (tid == 0) {
    // k == W: a beam's best continuation in the beam's place, the rest in the free places in order.
    unsigned used[LOGKV_BEAM_MAX_K / 32] = {0, 0, 0, 0};
    for (int i = 0; i < found; ++i) {
      const int w = bflat[i] / a.V;
      const bool first = !(used[w >> 5] >> (w & 31) & 1);
      place[i] = first ? (short)w : (short)-1;
      used[w >> 5] |= 1u << (w & 31);
    }
    int next = 0;
    for (int i = 0; i < k; ++i) {
      if (i < found && place[i] >= 0) continue;
      while (used[next >> 5] >> (next & 31) & 1) ++next;
      place[i] = (short)next++;
    }
  }
  __syncthreads();
  for (int i = tid; i < k; i += kBeamThreads) {
    const int p = place[i];
    const size_t o = (size_t)n * k + p;
    const bool is = i < found;
    const U64 q = is ? best[i] : 0ull;
    a.out_scores[o] = is ? (float)__longlong_as_double((long long)(q >> 63 ? q & 0x7fffffffffffffffull : ~q)) : -INFINITY;
    a.out_rows[o] = (long long)n * W + (is ? bflat[i] / a.V : min(p, W - 1));
    a.out_tokens[o] = is ? bflat[i] % a.V : 0;
  }
}

// ---------------------------------------------------------------- host side
static int beam_chunks(int vocab, int esize) {   // the row may start up to 15 bytes behind a boundary
  const long long per = kBeamThreads * kBeamVecs * (16 / esize);
  return (int)((vocab + 16 / esize - 1 + per - 1) / per);
}
// Slices of a beam: six CTAs per SM over all beams, a chunk each at least.
static int beam_slices(long long rows, int chunks) {
  return (int)std::max(1LL, std::min<long long>(chunks, (888 + rows - 1) / rows));
}

static bool beam_ok(int requests, int width, int vocab, int k) {
  return requests >= 1 && width >= 1 && width <= LOGKV_BEAM_MAX_WIDTH && vocab >= 1 && k >= 1 &&
         k <= LOGKV_BEAM_MAX_K && (long long)width * vocab < (1LL << 31) - 32 && k <= (long long)width * vocab &&
         (long long)requests * width <= 65535;
}

}  // namespace logkv

using namespace logkv;

extern "C" {

LOGKV_API size_t logkv_beam_workspace_bytes(int32_t requests, int32_t width, int32_t vocab, int32_t k) {
  if (!beam_ok(requests, width, vocab, k)) return 0;
  // Of either logits type: bf16 has no more chunks than float32.
  const size_t rows = (size_t)requests * width, lists = rows * beam_slices(rows, beam_chunks(vocab, 4));
  return lists * (sizeof(double) + sizeof(float)) + lists * k * (sizeof(float) + sizeof(int));
}

LOGKV_API int logkv_beam_select(const logkv_beam_args_t* x, void* workspace, size_t workspace_bytes, void* stream) {
  if (!x) return LOGKV_E_POINTER;
  if (x->dtype != LOGKV_DTYPE_F32 && x->dtype != LOGKV_DTYPE_BF16) return LOGKV_E_DTYPE;
  if (!beam_ok(x->requests, x->width, x->vocab, x->k) || (x->keep_places && x->k != x->width)) return LOGKV_E_SHAPE;
  auto at = [](const void* p, size_t n) { return p && (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  if (!at(x->logits, x->dtype == LOGKV_DTYPE_F32 ? 4 : 2) || !at(x->scores, 4) || !at(x->out_scores, 4) ||
      !at(x->out_rows, 8) || !at(x->out_tokens, 8) || !at(workspace, 8))
    return LOGKV_E_POINTER;
  if (workspace_bytes < logkv_beam_workspace_bytes(x->requests, x->width, x->vocab, x->k)) return LOGKV_E_WORKSPACE;
  const int rows = x->requests * x->width;
  BeamGeo a{};
  a.logits = x->logits;
  a.scores = x->scores;
  a.out_scores = x->out_scores;
  a.out_rows = reinterpret_cast<long long*>(x->out_rows);
  a.out_tokens = reinterpret_cast<long long*>(x->out_tokens);
  a.n_stride = x->n_stride;
  a.w_stride = x->w_stride;
  a.W = x->width;
  a.V = x->vocab;
  a.k = x->k;
  a.keep = x->keep_places;
  a.chunks = beam_chunks(x->vocab, x->dtype == LOGKV_DTYPE_F32 ? 4 : 2);
  a.S = beam_slices(rows, a.chunks);
  const size_t lists = (size_t)rows * a.S;
  a.sum = static_cast<double*>(workspace);
  a.top = reinterpret_cast<float*>(a.sum + lists);
  a.val = a.top + lists;
  a.idx = reinterpret_cast<int*>(a.val + lists * x->k);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (x->dtype == LOGKV_DTYPE_F32) launch_pdl(beam_slice_kernel<float>, dim3(a.S, rows), kBeamThreads, 0, st, a);
  else launch_pdl(beam_slice_kernel<__nv_bfloat16>, dim3(a.S, rows), kBeamThreads, 0, st, a);
  launch_pdl(beam_merge_kernel, dim3(x->requests), kBeamThreads, 0, st, a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? LOGKV_OK : (int)e;
}

}  // extern "C"
