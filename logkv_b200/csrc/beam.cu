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
//
// Bound by HBM at best: each logit is read once, 24 us for 32 x 16 beams x 151936 in bf16.  Measured 53.5 us there:
// 44 for B1 (31 for the walk, whose 7.7 instructions and one exponential a logit bound it, and the
// selections) and 10 for B2; 20 us for 29 x 5 x 50021 in float32, 11 for 4 x 32000.  The search bit by bit
// reads a slice 65 times: thousands of equal logits among a slice's k best (a finite mask over all but a few
// tokens) cost 3.8 ms at 32 x 16 x 151936, where a mask of -inf costs 49 us.
#include <algorithm>

#include "common.cuh"
#include "tcgen05.cuh"
#include "../../include/logkv_beam.h"

namespace logkv {

constexpr int kBeamThreads = 256;
constexpr int kBeamCand = 1024;    // gathered candidates at most
constexpr int kBeamVecs = 4;       // 16-byte vectors per thread and chunk
constexpr int kBeamGroups = 32;    // groups of chunks whose maxima a thread keeps
constexpr int kBeamHits = 1024;    // (thread, group) pairs that reach the threshold, at most

struct BeamGeo {
  const void* logits;
  const float* scores;
  float* out_scores;
  long long* out_rows;
  long long* out_tokens;
  long long n_stride, w_stride;
  int W, V, k, keep;
  int f32;        // logits are float32 (else bf16)
  int rows;       // beams in all
  int chunks;     // chunks (kBeamThreads x kBeamVecs vectors) of a beam's vocabulary
  int S;          // slices of a beam at most
  // Scratch per (request, beam, slice): the sum of 2^((x - top) e') and top; the k best logits, sorted.
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
  constexpr int N = 16 / sizeof(K);   // keys per shared-memory read
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
    int above = 0, same = 0;
#pragma unroll 4
    for (int g = 0; g < ng; g += N) {
      K q[N];
      *reinterpret_cast<uint4*>(q) = *reinterpret_cast<const uint4*>(gm + g);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        above += q[e] > me;
        same += q[e] == me;
      }
    }
    if (above < k && above + same >= k) *sh = me;   // equal maxima write the same value
  }
  __syncthreads();
  return *sh;
}

// Number of the n keys (16-byte aligned, an even number of places) that are above `me`.
__device__ __forceinline__ int keys_above(const unsigned long long* keys, int n, unsigned long long me) {
  int above = 0;
#pragma unroll 4
  for (int j = 0; j < n; j += 2) {
    const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(keys + j);
    above += q.x > me;
    above += q.y > me && j + 1 < n;
  }
  return above;
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

// Up to here a maximum's rounded offset max e' is off by at most 2^-4, so that the terms taken with it and the
// factor that puts them right are both near one.  (The error is half a unit of max e': 439 for logits masked
// with -1e10, where one of the two would be 0 and the other infinite.)  Beyond, the difference is taken first,
// an instruction more per two logits: 32 x 16 beams x 151936 take 56 us that way, 52 the first.
constexpr float kBeamNear = 1048576.f;   // 2^20

// The chunks of all beams are divided evenly among the CTAs, so a CTA's share may end in one beam and go
// on in the next; each part is a slice.  A slice is walked with the next chunks' loads in flight and no
// barrier in between: every thread keeps the running maximum and sum of its own terms, and the maximum
// of every group of chunks.  The threads' maxima give the threshold; the few (thread, group) pairs that
// reach it have their logits read again (from L2) and gathered.
template <typename T>
__global__ void __launch_bounds__(kBeamThreads, 4) beam_slice_kernel(BeamGeo a) {
  using U64 = unsigned long long;
  using Word = BeamWord<T>;
  constexpr int WN = Word::N, VN = 4 * WN, NV = kBeamVecs, NW = 4 * NV, CH = kBeamThreads * NV;
  __shared__ __align__(16) unsigned gm[kBeamThreads];
  __shared__ unsigned sh_t;
  __shared__ __align__(16) U64 cand[kBeamCand];
  __shared__ float tops[kBeamGroups][kBeamThreads];
  __shared__ float wmax[kBeamThreads / 32];
  __shared__ double wsum[kBeamThreads / 32];
  __shared__ int isum[kBeamThreads / 32];
  __shared__ int sh_n, sh_h;
  __shared__ unsigned short hits[kBeamHits];
  pdl_entry();
  const int tid = threadIdx.x, k = a.k;
  const long long all = (long long)a.rows * a.chunks, ctas = gridDim.x;
  const long long end = all * (blockIdx.x + 1) / ctas;
  long long at_chunk = all * blockIdx.x / ctas;
 next_slice:
  if (at_chunk >= end) return;
  const int rw = (int)(at_chunk / a.chunks), w = rw % a.W, n = rw / a.W;
  const int c0 = (int)(at_chunk - (long long)rw * a.chunks), c1 = (int)min((long long)a.chunks, c0 + (end - at_chunk));
  at_chunk += c1 - c0;
  // The row from the 16-byte boundary at or below its start: element e of it is logit e - lead.
  const T* row = static_cast<const T*>(a.logits) + n * a.n_stride + w * a.w_stride;
  const int lead = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  const T* base = row - lead;
  const uint4* vec = reinterpret_cast<const uint4*>(base);
  const int nvec = (a.V + lead + VN - 1) / VN;
  const int per = (c1 - c0 + kBeamGroups - 1) / kBeamGroups;   // chunks per group
  // The row's first and last vectors may hold a neighbour's logits: then they are left out here and their
  // own logits come after the walk, one by one, from the thread that would have had the vector.
  const int tail = nvec * VN - lead - a.V, lo = lead ? 1 : 0, hi = tail ? nvec - 1 : nvec;
  auto fetch = [&](int c, unsigned* x) {
    const int j0 = c * CH + tid;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      uint4 v = make_uint4(Word::kNone, Word::kNone, Word::kNone, Word::kNone);
      const int j = j0 + i * kBeamThreads;
      if (j >= lo && j < hi) v = __ldg(vec + j);
      x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
    }
  };
  float m = -INFINITY, s = 0.f, mg = -INFINITY;
  int left = per, group = 0;
  auto step = [&](const unsigned* x) {
    unsigned mx = x[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) mx = Word::max(mx, x[i]);
    const float mt = Word::top(mx);
    if (mt > m) {
      s = m == -INFINITY ? s : s * tc::ex2((m - mt) * kLog2e);   // s without a finite maximum: 0 or NaN
      m = mt;
    }
    mg = fmaxf(mg, mt);
    if (--left == 0) {
      tops[group++][tid] = mg;
      mg = -INFINITY;
      left = per;
    }
    const float ref = m == -INFINITY ? 0.f : m;
    const uint64_t e2 = tc::f2pack(kLog2e, kLog2e);
    uint64_t s2 = tc::f2pack(0.f, 0.f);
    float s0, s1;
    auto sum = [&](auto exponents) {
#pragma unroll
      for (int i = 0; i < NW; i += 2 / WN) {
        const float x0 = Word::get(x[i], 0), x1 = WN == 2 ? Word::get(x[i], 1) : Word::get(x[(i + 1) % NW], 0);
        float y0, y1;
        tc::f2unpack(exponents(tc::f2pack(x0, x1)), y0, y1);
        s2 = tc::fadd2(s2, tc::f2pack(tc::ex2(y0), tc::ex2(y1)));
      }
      tc::f2unpack(s2, s0, s1);
    };
    if (fabsf(ref) < kBeamNear) {
      // (x - ref) e' as one fused product with the offset rounded; the sum is put right below.
      const float off = ref * kLog2e;
      const uint64_t o2 = tc::f2pack(-off, -off);
      sum([&](uint64_t x2) { return tc::ffma2(x2, e2, o2); });
      s += (s0 + s1) * tc::ex2(fmaf(-ref, kLog2e, off));   // the offset's rounding error
    } else {   // the difference first: exact near ref, -inf (a term of 0) where it overflows
      const uint64_t r2 = tc::f2pack(-ref, -ref);
      sum([&](uint64_t x2) { return tc::fmul2(tc::fadd2(x2, r2), e2); });
      s += s0 + s1;
    }
  };
  unsigned xa[NW], xb[NW];
  fetch(c0, xa);
  if (c0 + 1 < c1) fetch(c0 + 1, xb);
  for (int c = c0; c < c1; c += 2) {
    step(xa);
    if (c + 2 < c1) fetch(c + 2, xa);
    if (c + 1 < c1) {
      step(xb);
      if (c + 3 < c1) fetch(c + 3, xb);
    }
  }
  if (left != per) tops[group][tid] = mg;
  auto own = [&](int j, auto use) {   // the row's logits in vector j, one by one
#pragma unroll 1
    for (int e = max(j * VN, lead); e < min((j + 1) * VN, lead + a.V); ++e) use((float)base[e], e - lead);
  };
  auto single = [&](int j) {
    const int c = j / CH;
    if (tid != j % kBeamThreads || c < c0 || c >= c1) return;
    float best = -INFINITY;
    own(j, [&](float f, int) {
      if (f > m) {
        s = m == -INFINITY ? s : s * tc::ex2((m - f) * kLog2e);
        m = f;
      }
      s += tc::ex2((f - (m == -INFINITY ? 0.f : m)) * kLog2e);
      best = fmaxf(best, f);
    });
    float& top = tops[(c - c0) / per][tid];
    top = fmaxf(top, best);
  };
  if (lead) single(0);
  if (tail && !(lead && nvec == 1)) single(nvec - 1);
  if (tid == 0) sh_n = sh_h = 0;
  // The slice's sum: the threads' maxima and float32 sums, joined in float64.
  const float mw = warp_max(m);
  if ((tid & 31) == 0) wmax[tid >> 5] = mw;
  const unsigned none = order32(-INFINITY);
  const unsigned t = max(group_threshold<unsigned>(order32(m), k, gm, &sh_t), none);   // its barriers publish wmax
  float top = wmax[0];
#pragma unroll
  for (int i = 1; i < kBeamThreads / 32; ++i) top = fmaxf(top, wmax[i]);
  double sd = m == -INFINITY ? (double)s : (double)s * exp2f((m - top) * kLog2e);
#pragma unroll
  for (int off = 16; off; off >>= 1) sd += __shfl_xor_sync(0xffffffffu, sd, off);
  if ((tid & 31) == 0) wsum[tid >> 5] = sd;
  // Gather the logits at or above the threshold (all above -inf when fewer than k groups hold any): the
  // (thread, group) pairs that reach it in a list, a warp to each, a lane to each of its logits.
  const float least = t == none ? -INFINITY : __uint_as_float(t & 0x80000000u ? t & 0x7fffffffu : ~t);
  for (int g = 0; g * per < c1 - c0; ++g) {
    const float f = tops[g][tid];
    if (f >= least && f > -INFINITY) {
      const int h = atomicAdd(&sh_h, 1);
      if (h < kBeamHits) hits[h] = (unsigned short)(g << 8 | tid);
    }
  }
  __syncthreads();
  // Four pairs of a warp at a time, so that their loads wait together.
  static_assert(NV * VN <= 32, "a lane per logit of a chunk");
  constexpr int WARPS = kBeamThreads / 32;
  const int nh = min(sh_h, kBeamHits), lane = tid & 31;
  for (int c = 0; c < per; ++c)
    for (int h0 = tid >> 5; h0 < nh; h0 += 4 * WARPS) {
      float f[4];
      int v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int h = h0 + i * WARPS, hit = h < nh ? hits[h] : 0, ch = c0 + (hit >> 8) * per + c;
        const int e = (ch * CH + lane / VN * kBeamThreads + (hit & 255)) * VN + lane % VN;
        v[i] = e - lead;
        f[i] = h < nh && ch < c1 && lane < NV * VN && v[i] >= 0 && v[i] < a.V ? (float)base[e] : -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (f[i] >= least && f[i] > -INFINITY) {
          const int at = atomicAdd(&sh_n, 1);
          if (at < kBeamCand) cand[at] = beam_key(f[i], v[i]);
        }
    }
  __syncthreads();
  int nc = sh_n;
  // The slice's place among its beam's: counted from the CTA that holds the beam's first chunk.
  const int slot = (int)(blockIdx.x - (((long long)rw * a.chunks + 1) * ctas - 1) / all);
  const size_t at = (size_t)rw * a.S + slot;
  if (tid == 0) {
    double total = 0.0;
    for (int i = 0; i < kBeamThreads / 32; ++i) total += wsum[i];
    a.sum[at] = total;
    a.top[at] = top;
  }
  if (nc > kBeamCand || sh_h > kBeamHits) {
    // More than the buffers hold: the k-th largest key bit by bit, the logits read again each time.
    auto visit = [&](auto take) {
      for (int c = c0; c < c1; ++c)
#pragma unroll 1
        for (int i = 0; i < NV; ++i) {
          const int j = c * CH + i * kBeamThreads + tid;
          if (j >= nvec) break;
          if (j < lo || j >= hi) {   // a ragged end, as in the walk
            own(j, [&](float f, int v) {
              if (f > -INFINITY) take(beam_key(f, v));
            });
            continue;
          }
          const uint4 q = __ldg(vec + j);
          const unsigned x[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int e = 0; e < VN; ++e) {
            const float f = Word::get(x[e / WN], e % WN);
            if (f > -INFINITY) take(beam_key(f, j * VN + e - lead));
          }
        }
    };
    U64 kt = 0;
    for (int bit = 63; bit >= 0; --bit) {
      const U64 test = kt | 1ull << bit;
      int cnt = 0;
      visit([&](U64 key) { cnt += key >= test; });
      if (block_sum(cnt, isum) >= k) kt = test;
    }
    if (tid == 0) sh_n = 0;
    __syncthreads();
    visit([&](U64 key) {
      if (key >= kt) cand[atomicAdd(&sh_n, 1)] = key;
    });
    __syncthreads();
    nc = k;
  }
  float* val = a.val + at * k;
  int* idx = a.idx + at * k;
  for (int i = tid; i < nc; i += kBeamThreads) {
    const U64 me = cand[i];
    const int above = keys_above(cand, nc, me);
    if (above < k) {
      val[above] = key_value(me);
      idx[above] = (int)(0xffffffffu - (unsigned)me);
    }
  }
  for (int i = nc + tid; i < k; i += kBeamThreads) idx[i] = -1;
  if (c1 == a.chunks) {   // the beam's last slice: the places behind it hold nothing
    for (int i = tid; i < (a.S - 1 - slot) * k; i += kBeamThreads) idx[k + i] = -1;
    for (int i = slot + 1 + tid; i < a.S; i += kBeamThreads) {
      a.sum[(size_t)rw * a.S + i] = 0.0;
      a.top[(size_t)rw * a.S + i] = -INFINITY;
    }
  }
  __syncthreads();   // before the next slice uses the shared memory again
  goto next_slice;
}

// ---------------------------------------------------------------- B2
// The candidates in rounds of up to kBeamRound, the k best so far among each round's.
constexpr int kBeamRound = 2048, kBeamEach = kBeamRound / kBeamThreads;

// The slices' sums are off by up to 1.2e-7 relative (measured over alignments, slices and vocabularies of 37 to
// 151936), so continuations of different beams whose scores are further apart than this are in their order
// (those of one beam always are).  Beams with closer ones, equal beams above all, have their logits summed in
// float64, in an order that is the same for every alignment, and are merged again: 115 us a beam of 151936.
constexpr double kBeamClose = 1.0 / (1 << 21);

// What two roundings of a beam's scores to float64 may differ by, beside that.  (From 1e17 on the maximum
// swallows the logarithm, and there is nothing to round.)
__device__ __forceinline__ double beam_wobble(float peak) {
  const double p = fabs((double)peak);
  return p < 1e17 ? p * (1.0 / (1ull << 51)) : 0.0;
}
__device__ __forceinline__ double key_score(unsigned long long q) {
  return __longlong_as_double((long long)(q >> 63 ? q & 0x7fffffffffffffffull : ~q));
}

// The thread's share of a row's sum of exponentials in float64 (not inlined: its registers stay out of the merge).
template <typename T>
__device__ __noinline__ double beam_sum(const T* row, unsigned V, double top) {
  double sum = 0.0;
  for (unsigned j0 = threadIdx.x; j0 < V; j0 += 8 * kBeamThreads) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = j0 + i * kBeamThreads < V ? (float)row[j0 + i * kBeamThreads] : -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += exp((double)x[i] - top);
  }
  return sum;
}

__global__ void __launch_bounds__(kBeamThreads) beam_merge_kernel(BeamGeo a) {
  using U64 = unsigned long long;
  __shared__ __align__(16) U64 gm[kBeamThreads];
  __shared__ U64 sh_t;
  __shared__ __align__(16) U64 cand[kBeamCand];
  __shared__ int cidx[kBeamCand];
  __shared__ double lse[LOGKV_BEAM_MAX_WIDTH];
  __shared__ float prior[LOGKV_BEAM_MAX_WIDTH], peak[LOGKV_BEAM_MAX_WIDTH];
  __shared__ unsigned close_beams[LOGKV_BEAM_MAX_WIDTH / 32];
  __shared__ double wsum[kBeamThreads / 32];
  __shared__ int isum[kBeamThreads / 32];
  __shared__ int sh_n;
  __shared__ U64 best[LOGKV_BEAM_MAX_K];
  __shared__ int bflat[LOGKV_BEAM_MAX_K];
  __shared__ short place[LOGKV_BEAM_MAX_K];
  pdl_entry();
  const int tid = threadIdx.x, n = blockIdx.x, W = a.W, S = a.S, k = a.k;
  const float* val = a.val + (size_t)n * W * S * k;
  const int* idx = a.idx + (size_t)n * W * S * k;
  // Candidate i is place i / L of list i % L, so that every group of threads sees a mix of lists.
  const int L = W * S, all = L * k;
  // The first round's candidates are on their way while the beams' sums are joined.
  float v[kBeamEach];
  int vi[kBeamEach];
  auto fetch = [&](int from, int upto) {
#pragma unroll
    for (int i = 0; i < kBeamEach; ++i) {
      const int at = from + i * kBeamThreads + tid;
      const int where = at % L * k + at / L;
      vi[i] = at < upto ? idx[where] : -1;
      v[i] = at < upto ? val[where] : 0.f;
    }
  };
  int upto = min(all, kBeamRound);
  fetch(0, upto);
  // log sum exp of each beam in float64; NaN for a beam that offers nothing.  A lane to a slice: 2 to 32
  // lanes to a beam.
  int lanes = 2;
  while (lanes < S && lanes < 32) lanes *= 2;
  bool wobbles = false;
  for (int w0 = 0; w0 < W; w0 += kBeamThreads / lanes) {
    const int w = w0 + tid / lanes, first = tid % lanes;
    const size_t at = (size_t)(n * W + min(w, W - 1)) * S;
    float m = -INFINITY;
    for (int q = first; q < S; q += lanes) m = fmaxf(m, a.sum[at + q] > 0.0 ? a.top[at + q] : -INFINITY);
    for (int off = 1; off < lanes; off *= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    double s = 0.0;
    for (int q = first; q < S; q += lanes)
      if (a.sum[at + q] != 0.0) s += a.sum[at + q] * exp2f((a.top[at + q] - m) * kLog2e);   // a NaN stays
    for (int off = 1; off < lanes; off *= 2) s += __shfl_xor_sync(0xffffffffu, s, off);
    if (first == 0 && w < W) {
      wobbles |= beam_wobble(m) > kBeamClose;
      const float r = a.scores[n * W + w];
      const double z = (double)m + log2(s) / (double)kLog2e;
      lse[w] = isfinite(r) && isfinite(z) ? z : nan("");
      prior[w] = r;
      peak[w] = m;
    }
  }
  wobbles = __syncthreads_or(wobbles);
  bool exact = W == 1;
  int found;
  // Keys (score, 0 for none) and flat indices of the candidates fetched.
  U64 key[kBeamEach];
  int flat[kBeamEach];
  auto rate = [&](int from) {
#pragma unroll
    for (int i = 0; i < kBeamEach; ++i) {
      key[i] = 0;
      flat[i] = 0x7fffffff;
      if (vi[i] >= 0) {
        const int w = (from + i * kBeamThreads + tid) % L / S;
        if (!isnan(lse[w])) {
          key[i] = order64((double)prior[w] + ((double)v[i] - lse[w]));
          flat[i] = w * a.V + vi[i];
        }
      }
    }
  };
 merge:
  found = 0;
  for (int from = 0; from < all;) {
    rate(from);
    U64 mine = 0;
#pragma unroll
    for (int i = 0; i < kBeamEach; ++i) {
      const int at = from + i * kBeamThreads + tid;
      if (at >= upto && at - upto < found) {   // the best so far take the last places
        key[i] = best[at - upto];
        flat[i] = bflat[at - upto];
      }
      mine = key[i] > mine ? key[i] : mine;
    }
    if (tid == 0) sh_n = 0;
    U64 t = group_threshold<U64>(mine, k, gm, &sh_t);
    t = t ? t : 1;
    const int next = upto, step = min(all, upto + kBeamRound - k);
    if (next < all) fetch(next, step);
    int cnt = 0;
#pragma unroll
    for (int i = 0; i < kBeamEach; ++i) cnt += key[i] >= t;
    int tf = 0x7fffffff;   // flat indices taken at the threshold itself
    if (block_sum(cnt, isum) > kBeamCand) {
      t = 0;
      for (int bit = 63; bit >= 0; --bit) {
        const U64 test = t | 1ull << bit;
        cnt = 0;
#pragma unroll
        for (int i = 0; i < kBeamEach; ++i) cnt += key[i] >= test;
        if (block_sum(cnt, isum) >= k) t = test;
      }
      cnt = 0;
#pragma unroll
      for (int i = 0; i < kBeamEach; ++i) cnt += key[i] > t;
      const int need = k - block_sum(cnt, isum);
      int low = 0;   // the `need` lowest flat indices among the ties: flat <= low
      for (int bit = 30; bit >= 0; --bit) {
        const int test = low | 1 << bit;
        cnt = 0;
#pragma unroll
        for (int i = 0; i < kBeamEach; ++i) cnt += key[i] == t && flat[i] < test;
        if (block_sum(cnt, isum) < need) low = test;
      }
      tf = low;
    }
#pragma unroll
    for (int i = 0; i < kBeamEach; ++i)
      if (key[i] > t || (key[i] == t && flat[i] <= tf)) {
        const int at = atomicAdd(&sh_n, 1);
        cand[at] = key[i];
        cidx[at] = flat[i];
      }
    __syncthreads();
    const int nc = sh_n;
    for (int i = tid; i < nc; i += kBeamThreads) {
      const U64 me = cand[i];
      const int mf = cidx[i];
      int above = keys_above(cand, nc, me);
      if (above < k)   // equal scores: the lower flat index first
        for (int j = 0; j < nc; ++j) above += cand[j] == me && cidx[j] < mf;
      if (above < k) {
        best[above] = me;
        bflat[above] = mf;
      }
    }
    found = min(nc, k);
    from = next;
    upto = step;
    __syncthreads();
  }
  if (!exact) {
    // Beams that have a continuation close to another beam's, among those chosen or at their border.
    if (tid < LOGKV_BEAM_MAX_WIDTH / 32) close_beams[tid] = 0;
    __syncthreads();
    auto mark = [&](int w) { atomicOr(&close_beams[w >> 5], 1u << (w & 31)); };
    auto compare = [&](double higher, int w, double lower, int x) {
      if (w != x && higher - lower <= kBeamClose + beam_wobble(peak[w]) + beam_wobble(peak[x])) {
        mark(w);
        mark(x);
      }
    };
    if (tid + 1 < found) compare(key_score(best[tid]), bflat[tid] / a.V, key_score(best[tid + 1]), bflat[tid + 1] / a.V);
    if (found == k) {
      const U64 last = best[k - 1];
      const int last_flat = bflat[k - 1];
      const double border = key_score(last);
      for (int from = 0; from < all; from += kBeamRound) {
        if (all > kBeamRound) {   // else they are still there
          fetch(from, min(all, from + kBeamRound));
          rate(from);
        }
#pragma unroll
        for (int i = 0; i < kBeamEach; ++i) {
          const bool left = key[i] && (key[i] < last || (key[i] == last && flat[i] > last_flat));
          const double y = key_score(key[i]);
          if (left && (wobbles || border - y <= 3 * kBeamClose)) compare(border, last_flat / a.V, y, flat[i] / a.V);
        }
      }
    }
    __syncthreads();
    unsigned any = 0;
    for (int i = 0; i < LOGKV_BEAM_MAX_WIDTH / 32; ++i) any |= close_beams[i];
    if (any) {
      for (int w = 0; w < W; ++w) {
        if (!(close_beams[w >> 5] >> (w & 31) & 1)) continue;
        const long long row = n * a.n_stride + w * a.w_stride;
        const double top = peak[w];
        double sum = a.f32 ? beam_sum(static_cast<const float*>(a.logits) + row, a.V, top)
                           : beam_sum(static_cast<const __nv_bfloat16*>(a.logits) + row, a.V, top);
#pragma unroll
        for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        if ((tid & 31) == 0) wsum[tid >> 5] = sum;
        __syncthreads();
        if (tid == 0) {
          double total = 0.0;
          for (int i = 0; i < kBeamThreads / 32; ++i) total += wsum[i];
          lse[w] = top + log(total);
        }
        __syncthreads();
      }
      exact = true;
      upto = min(all, kBeamRound);
      fetch(0, upto);
      goto merge;
    }
  }
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
    a.out_scores[o] = is ? (float)key_score(best[i]) : -INFINITY;
    a.out_rows[o] = (long long)n * W + (is ? bflat[i] / a.V : min(p, W - 1));
    a.out_tokens[o] = is ? bflat[i] % a.V : 0;
  }
}

// ---------------------------------------------------------------- host side
static int beam_chunks(int vocab, int esize) {   // the row may start up to 15 bytes behind a boundary
  const long long per = kBeamThreads * kBeamVecs * (16 / esize);
  return (int)((vocab + 16 / esize - 1 + per - 1) / per);
}
// CTAs: four per SM (as many as run at once), a chunk each at least; a beam's slices at most.
static long long beam_ctas(long long rows, int chunks) { return std::min<long long>(rows * chunks, 592); }
static int beam_slices(long long rows, int chunks) {
  const long long each = rows * chunks / beam_ctas(rows, chunks);
  return (int)((chunks - 1 + each - 1) / each + 1);
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
  // Of either logits type.
  const size_t rows = (size_t)requests * width;
  const size_t lists = rows * std::max(beam_slices(rows, beam_chunks(vocab, 4)), beam_slices(rows, beam_chunks(vocab, 2)));
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
  a.f32 = x->dtype == LOGKV_DTYPE_F32;
  a.chunks = beam_chunks(x->vocab, x->dtype == LOGKV_DTYPE_F32 ? 4 : 2);
  a.rows = rows;
  a.S = beam_slices(rows, a.chunks);
  const size_t lists = (size_t)rows * a.S;
  a.sum = static_cast<double*>(workspace);
  a.top = reinterpret_cast<float*>(a.sum + lists);
  a.val = a.top + lists;
  a.idx = reinterpret_cast<int*>(a.val + lists * x->k);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)beam_ctas(rows, a.chunks));
  if (x->dtype == LOGKV_DTYPE_F32) launch_pdl(beam_slice_kernel<float>, grid, kBeamThreads, 0, st, a);
  else launch_pdl(beam_slice_kernel<__nv_bfloat16>, grid, kBeamThreads, 0, st, a);
  launch_pdl(beam_merge_kernel, dim3(x->requests), kBeamThreads, 0, st, a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? LOGKV_OK : (int)e;
}

}  // extern "C"
