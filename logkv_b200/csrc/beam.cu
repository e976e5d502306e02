// Beam search's selection over beams and vocabulary (C ABI in include/logkv_beam.h).
//
//   B1 beam_slice_kernel  one CTA per slice of a beam's vocabulary: one read of the logits into
//                          registers gives the slice's sum of exponentials and its k best logits;
//   B2 beam_merge_kernel  one CTA per request: every beam's log-sum-exp from its slices, then the k
//                          best of all slices' lists by score.
//
// Both choose the k best the same way.  The threads are put into at least 2 k groups; the k-th
// largest of the groups' maxima has at least k elements at or above it and, unless the values are
// very uneven, not many more; those are gathered and ranked by counting.  When too many are at or
// above it (ties), the k-th largest key is found bit by bit instead.  Keys are (value, lower index
// first), so the choice is unique whatever the order of the gathering.
#include <algorithm>

#include "common.cuh"
#include "../../include/logkv_beam.h"

namespace logkv {

constexpr int kBeamThreads = 512;
constexpr int kBeamCand = 1024;    // gathered candidates at most

struct BeamGeo {
  const void* logits;
  const float* scores;
  float* out_scores;
  long long* out_rows;
  long long* out_tokens;
  long long n_stride, w_stride;
  int W, V, k, S, keep;
  int slice;      // vectors per slice
  // Scratch: per (request, beam, slice) the sum of exp(x - top) and top; per request [k][W * S] lists.
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

// Threads per group: 64 groups or more, at least 2 k (256 groups for the largest k).
__device__ __forceinline__ int group_size(int k) { return k <= 32 ? 8 : k <= 64 ? 4 : 2; }

// The k-th largest of the groups' maxima (0 when fewer groups hold anything).  `gm`: one entry per group.
template <typename K>
__device__ __forceinline__ K group_threshold(K mine, int k, K* gm, K* sh) {
  const int gs = group_size(k), ng = kBeamThreads / gs, tid = threadIdx.x;
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
    for (int g = 0; g < ng; ++g) above += gm[g] > me || (gm[g] == me && g < tid);
    if (above == k - 1) *sh = me;
  }
  __syncthreads();
  return *sh;
}

// ---------------------------------------------------------------- B1
template <typename T>
struct BeamVec;
template <>
struct BeamVec<float> {
  static constexpr int N = 4;
  __device__ __forceinline__ static void unpack(const uint4& u, float* x) {
    x[0] = __uint_as_float(u.x);
    x[1] = __uint_as_float(u.y);
    x[2] = __uint_as_float(u.z);
    x[3] = __uint_as_float(u.w);
  }
};
template <>
struct BeamVec<__nv_bfloat16> {
  static constexpr int N = 8;
  __device__ __forceinline__ static void unpack(const uint4& u, float* x) {
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};

// E logits per thread.
template <typename T, int E>
__global__ void __launch_bounds__(kBeamThreads) beam_slice_kernel(BeamGeo a) {
  constexpr int VN = BeamVec<T>::N, NV = E / VN;
  __shared__ unsigned gm[kBeamThreads / 2];
  __shared__ unsigned sh_t;
  __shared__ unsigned long long cand[kBeamCand];
  __shared__ float wmax[kBeamThreads / 32];
  __shared__ double wsum[kBeamThreads / 32];
  __shared__ int isum[kBeamThreads / 32];
  __shared__ int sh_n;
  pdl_entry();
  const int tid = threadIdx.x, slice = blockIdx.x, w = blockIdx.y % a.W, n = blockIdx.y / a.W;
  // The row from the 16-byte boundary at or below its start: element e of it is logit e - lead.
  const T* row = static_cast<const T*>(a.logits) + n * a.n_stride + w * a.w_stride;
  const int lead = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  const uint4* vec = reinterpret_cast<const uint4*>(row - lead);
  const int nvec = (a.V + lead + VN - 1) / VN;
  const int v0 = slice * a.slice;
  uint4 raw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = v0 + i * kBeamThreads + tid;
    if (j < nvec) raw[i] = __ldcs(vec + j);
  }
  float x[E];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = v0 + i * kBeamThreads + tid;
    if (j < nvec) {
      BeamVec<T>::unpack(raw[i], x + i * VN);
      if (j == 0 || j == nvec - 1) {
#pragma unroll
        for (int e = 0; e < VN; ++e) {
          const int v = j * VN + e - lead;
          if (v < 0 || v >= a.V) x[i * VN + e] = -INFINITY;
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < VN; ++e) x[i * VN + e] = -INFINITY;
    }
  }
  float mt = -INFINITY;
#pragma unroll
  for (int e = 0; e < E; ++e) mt = fmaxf(mt, x[e]);
  const float mw = warp_max(mt);
  if ((tid & 31) == 0) wmax[tid >> 5] = mw;
  // The threshold's barriers also publish wmax.
  const unsigned none = order32(-INFINITY);
  const unsigned t = max(group_threshold<unsigned>(order32(mt), a.k, gm, &sh_t), none + 1);
  float m = wmax[0];
#pragma unroll
  for (int i = 1; i < kBeamThreads / 32; ++i) m = fmaxf(m, wmax[i]);
  // Sum of exp(x - m): the difference and the product with log2 e (in two parts, so that its own
  // rounding is no common factor) are off by half a unit each, at random over the terms; the float32
  // sums of a thread's terms are joined in float64.  m = 0 for a slice without a finite logit.
  if (m == -INFINITY) m = 0.f;
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float d = x[e] - m;
    s += exp2f(fmaf(d, 1.44269502f, d * 1.92596300e-8f));
  }
  double sd = s;
#pragma unroll
  for (int off = 16; off; off >>= 1) sd += __shfl_xor_sync(0xffffffffu, sd, off);
  if ((tid & 31) == 0) wsum[tid >> 5] = sd;
  if (tid == 0) sh_n = 0;
  __syncthreads();
  const size_t at = (size_t)blockIdx.y * a.S + slice;
  if (tid == 0) {
    double total = 0.0;
    for (int i = 0; i < kBeamThreads / 32; ++i) total += wsum[i];
    a.sum[at] = total;
    a.top[at] = m;
  }
  // Elements at or above the threshold (all numbers above -inf; NaN is below by the comparison).
  int mine = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) mine += x[e] > -INFINITY && order32(x[e]) >= t;
  const int total = block_sum(mine, isum);
  // Key: value, then the lower place in the slice.
  auto key = [&](int e) {
    const int local = (e / VN * kBeamThreads + tid) * VN + e % VN;
    return x[e] > -INFINITY ? (unsigned long long)order32(x[e]) << 14 | (16383 - local) : 0ull;
  };
  static_assert(E * kBeamThreads <= 16384, "place in a slice");
  unsigned long long kt = (unsigned long long)t << 14;
  if (total > kBeamCand) {
    kt = 0;
    for (int bit = 45; bit >= 0; --bit) {
      const unsigned long long test = kt | 1ull << bit;
      int cnt = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) cnt += key(e) >= test;
      if (block_sum(cnt, isum) >= a.k) kt = test;
    }
  }
  if (mine) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const unsigned long long q = key(e);
      if (q >= kt && q) cand[atomicAdd(&sh_n, 1)] = q;
    }
  }
  __syncthreads();
  const int nc = sh_n, L = a.W * a.S;
  float* val = a.val + (size_t)n * a.k * L + w * a.S + slice;
  int* idx = a.idx + (size_t)n * a.k * L + w * a.S + slice;
  for (int i = tid; i < nc; i += kBeamThreads) {
    const unsigned long long me = cand[i];
    int above = 0;
    for (int j = 0; j < nc; ++j) above += cand[j] > me;
    if (above < a.k) {
      const unsigned o = (unsigned)(me >> 14);
      val[(size_t)above * L] = __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
      idx[(size_t)above * L] = v0 * VN + (16383 - (int)(me & 16383)) - lead;
    }
  }
  for (int i = nc + tid; i < a.k; i += kBeamThreads) idx[(size_t)i * L] = -1;
}

// ---------------------------------------------------------------- B2
__global__ void __launch_bounds__(kBeamThreads) beam_merge_kernel(BeamGeo a) {
  using U64 = unsigned long long;
  __shared__ U64 gm[kBeamThreads / 2];
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
      if (si != 0.0) s += si * exp((double)a.top[at + i] - (double)m);   // a NaN stays
    }
#pragma unroll
    for (int off = 16; off; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    if (lane == 0) {
      const float r = a.scores[n * W + w];
      const double z = log(s) + (double)m;
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
// Slices: 16384 logits per CTA (32 per thread), less while the rows alone leave SMs idle.
static int beam_elems(long long rows, int vocab) {
  int e = 32;
  while (e > 8 && rows * ((vocab + 8 + e * kBeamThreads - 1) / (e * kBeamThreads)) < 296) e /= 2;
  return e;
}
// (a slice more than V needs when the row's start is not aligned)
static int beam_slices(int vocab, int elems) { return (vocab + 8 + elems * kBeamThreads - 1) / (elems * kBeamThreads); }

static bool beam_ok(int requests, int width, int vocab, int k) {
  return requests >= 1 && width >= 1 && width <= LOGKV_BEAM_MAX_WIDTH && vocab >= 1 && k >= 1 &&
         k <= LOGKV_BEAM_MAX_K && (long long)width * vocab < (1LL << 31) - 32 && k <= (long long)width * vocab &&
         (long long)requests * width <= 65535;
}

template <typename T>
static void launch_slices(const BeamGeo& a, int elems, int rows, cudaStream_t st) {
  const dim3 grid(a.S, rows);
  if (elems == 32) launch_pdl(beam_slice_kernel<T, 32>, grid, kBeamThreads, 0, st, a);
  else if (elems == 16) launch_pdl(beam_slice_kernel<T, 16>, grid, kBeamThreads, 0, st, a);
  else launch_pdl(beam_slice_kernel<T, 8>, grid, kBeamThreads, 0, st, a);
}

}  // namespace logkv

using namespace logkv;

extern "C" {

LOGKV_API size_t logkv_beam_workspace_bytes(int32_t requests, int32_t width, int32_t vocab, int32_t k) {
  if (!beam_ok(requests, width, vocab, k)) return 0;
  const size_t rows = (size_t)requests * width, lists = rows * beam_slices(vocab, beam_elems(rows, vocab));
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
  const int rows = x->requests * x->width, elems = beam_elems(rows, x->vocab);
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
  a.S = beam_slices(x->vocab, elems);
  a.slice = elems * kBeamThreads / (x->dtype == LOGKV_DTYPE_F32 ? 4 : 8);
  const size_t lists = (size_t)rows * a.S;
  a.sum = static_cast<double*>(workspace);
  a.top = reinterpret_cast<float*>(a.sum + lists);
  a.val = a.top + lists;
  a.idx = reinterpret_cast<int*>(a.val + lists * x->k);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (x->dtype == LOGKV_DTYPE_F32) launch_slices<float>(a, elems, rows, st);
  else launch_slices<__nv_bfloat16>(a, elems, rows, st);
  launch_pdl(beam_merge_kernel, dim3(x->requests), kBeamThreads, 0, st, a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? LOGKV_OK : (int)e;
}

}  // extern "C"
