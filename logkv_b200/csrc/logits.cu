// Penalties of repeated tokens, biases and grammar masks on next-token logits (C ABI in include/logkv_logits.h).
//
// Bound by HBM: every logit is read once and written once, the mask's bits are read once; below a few MB by the
// launch and one slice's latency.
//
// A CTA takes one slice of one row: its threads ask for the slice's logits first (PER 16-byte vectors each,
// kept in registers), and while those come scan the row's history for tokens of the slice.  Touched tokens are bits
// of a bitmap with a counter each in shared memory, so that a vector without a touched bit costs one byte of
// shared memory and is written back as it was read.  Counters are integers: the order of the scan does not show.
#include <algorithm>

#include "common.cuh"
#include "../../include/logkv_logits.h"

namespace logkv {

constexpr int kLogitsThreads = 256;
constexpr unsigned kSeen = 0x80000000u;   // counter bit of a token that the prompt holds

__device__ __forceinline__ long long load_int(const void* p, int wide, long long i) {
  return wide ? static_cast<const long long*>(p)[i] : (long long)static_cast<const int32_t*>(p)[i];
}

// Bits of tokens v .. v + n - 1 (n <= 8) of a row's mask, those of tokens past the vocabulary unset.
__device__ __forceinline__ unsigned mask_bits(const int32_t* mask, int v, int n, int vocab) {
  const int w0 = v >> 5, w1 = min(v + n - 1, vocab - 1) >> 5;
  const unsigned lo = (unsigned)mask[w0], hi = w1 != w0 ? (unsigned)mask[w1] : 0u;
  return __funnelshift_r(lo, hi, v & 31);
}

// Tokens of a row's history that lie in [begin, end), four loads in flight per thread: visit(index, token).
template <typename Visit>
__device__ __forceinline__ void visit_history(const logkv_logits_args_t& a, int r, int length, int begin, int end,
                                              Visit visit) {
  const long long h0 = (long long)r * a.history_stride;
  for (int i0 = threadIdx.x; i0 < length; i0 += 4 * kLogitsThreads) {
    long long v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + k * kLogitsThreads;
      v[k] = i < length ? load_int(a.history, a.history_wide, h0 + i) : -1;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (v[k] >= begin && v[k] < end) visit(i0 + k * kLogitsThreads, (int)v[k]);
  }
}

template <typename T, int PER>
__global__ void __launch_bounds__(kLogitsThreads) adjust_logits_kernel(logkv_logits_args_t a) {
  constexpr int VN = 16 / (int)sizeof(T), SLICE = kLogitsThreads * PER * VN;
  constexpr int BIAS = LOGKV_LOGITS_MAX_BIAS / kLogitsThreads;   // bias entries per thread
  extern __shared__ unsigned count[];                                   // [SLICE] where there is a history
  __shared__ unsigned touched[SLICE / 32];
  int* bt = reinterpret_cast<int*>(count + (a.history ? SLICE : 0));    // [bias_count] tokens, -1: not this slice's
  float* bv = reinterpret_cast<float*>(bt + a.bias_count);              // [bias_count] biases
  pdl_entry();
  const int tid = threadIdx.x, r = blockIdx.y, n = r / a.width, w = r % a.width;
  const T* x = static_cast<const T*>(a.logits) + n * a.n_stride + w * a.w_stride;
  T* y = static_cast<T*>(a.out) + n * a.out_n_stride + w * a.out_w_stride;
  // Slices start where the output's 16-byte vectors do: vector j of this one is tokens v0 + j VN and on.
  const int mis = (int)((reinterpret_cast<uintptr_t>(y) & 15) / sizeof(T));
  const int v0 = blockIdx.x * SLICE - mis, begin = max(v0, 0), end = min(a.vocab, v0 + SLICE);
  if (begin >= end) return;
  const bool shifted = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T)) != mis;

  uint4 raw[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int v = v0 + (tid + i * kLogitsThreads) * VN;
    raw[i] = make_uint4(0u, 0u, 0u, 0u);
    if (v >= begin && v + VN <= end) {
      if (!shifted) {
        raw[i] = *reinterpret_cast<const uint4*>(x + v);
      } else {
        // The logits' rows lie at another offset than the output's: four words, or, for bf16 at an odd element,
        // its two ends and three words.
        const uintptr_t at = reinterpret_cast<uintptr_t>(x + v);
        if (!(at & 3)) {
          const unsigned* s = reinterpret_cast<const unsigned*>(at);
          raw[i] = make_uint4(s[0], s[1], s[2], s[3]);
        } else {
          const unsigned short* e = reinterpret_cast<const unsigned short*>(at);
          const unsigned* s = reinterpret_cast<const unsigned*>(at + 2);
          const unsigned w0 = e[0], w1 = s[0], w2 = s[1], w3 = s[2], w4 = e[7];
          raw[i] = make_uint4(w0 | w1 << 16, __funnelshift_r(w1, w2, 16), __funnelshift_r(w2, w3, 16),
                              w3 >> 16 | w4 << 16);
        }
      }
    } else {   // a row's ragged end: element by element
      T* e = reinterpret_cast<T*>(&raw[i]);
#pragma unroll
      for (int j = 0; j < VN; ++j)
        if (v + j >= begin && v + j < end) e[j] = x[v + j];
    }
  }

  const float rep = a.repetitions ? a.repetitions[r] : a.repetition;
  const float pres = a.presences ? a.presences[r] : a.presence, freq = a.frequencies ? a.frequencies[r] : a.frequency;
  if (a.history) {
    const long long len = a.lengths ? load_int(a.lengths, a.lengths_wide, r) : a.length;
    const int length = (int)max(0LL, min(len, (long long)a.history_len));
    const long long pro = a.prompts ? load_int(a.prompts, a.prompts_wide, r) : a.prompt;
    const int prompt = (int)max(0LL, min(pro, (long long)length));
    for (int i = tid; i < SLICE / 32; i += kLogitsThreads) touched[i] = 0u;
    __syncthreads();
    visit_history(a, r, length, begin, end, [&](int, int v) {
      count[v - v0] = 0u;   // the same value from every thread that meets the token
      atomicOr(&touched[(v - v0) >> 5], 1u << ((v - v0) & 31));
    });
    __syncthreads();
    visit_history(a, r, length, begin, end, [&](int i, int v) {
      if (i < prompt) atomicOr(&count[v - v0], kSeen);
      else atomicAdd(&count[v - v0], 1u);
    });
  }
  for (int i = tid; i < a.bias_count; i += kLogitsThreads) {
    const long long v = load_int(a.bias_tokens, a.bias_wide, r * a.bias_tokens_stride + i);
    bt[i] = v >= begin && v < end ? (int)v : -1;
    bv[i] = a.bias_values[r * a.bias_values_stride + i];
  }
  if (a.history || a.bias_count) __syncthreads();

  const int32_t* mask = a.mask ? a.mask + r * a.mask_stride : nullptr;
  auto adjust = [&](float z, unsigned c) {
    z = z > 0.f ? __fdiv_rn(z, rep) : z * rep;
    const unsigned k = c & ~kSeen;
    return k ? z - fmaf(freq, (float)k, pres) : z;
  };
  // Biased tokens are few: the thread of a token's first entry works out its value, and puts it over the slice's
  // own once that is written.
  float bz[BIAS];
  bool put[BIAS];
#pragma unroll
  for (int k = 0; k < BIAS; ++k) {
    const int i = tid + k * kLogitsThreads, v = i < a.bias_count ? bt[i] : -1;
    bool first = v >= 0;
    for (int j = 0; j < i && first; ++j) first = bt[j] != v;
    put[k] = first;
    bz[k] = 0.f;
    if (!first) continue;
    float sum = bv[i];
    for (int j = i + 1; j < a.bias_count; ++j)
      if (bt[j] == v) sum += bv[j];
    float z = Elem<T>::load(x + v);
    const int l = v - v0;
    if (a.history && touched[l >> 5] >> (l & 31) & 1) z = adjust(z, count[l]);
    z += sum;
    bz[k] = mask && !(mask_bits(mask, v, 1, a.vocab) & 1) ? -INFINITY : z;
  }
  if (a.bias_count) __syncthreads();   // in place: every biased logit is read before the slice is written

#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int l = (tid + i * kLogitsThreads) * VN, v = v0 + l;
    if (v >= end || v + VN <= begin) continue;
    T* e = reinterpret_cast<T*>(&raw[i]);
    if (a.history) {
      const unsigned t = touched[l >> 5] >> (l & 31) & ((1u << VN) - 1);
      if (t) {
#pragma unroll
        for (int j = 0; j < VN; ++j)
          if (t >> j & 1) Elem<T>::store(&e[j], adjust(Elem<T>::load(&e[j]), count[l + j]));
      }
    }
    if (mask) {
      const int s = max(v, begin);
      const unsigned m = mask_bits(mask, s, VN, a.vocab) << (s - v);
      unsigned* word = reinterpret_cast<unsigned*>(&raw[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (VN == 4)
          word[j] = m >> j & 1 ? word[j] : 0xff800000u;
        else
          word[j] = (m >> (2 * j) & 1 ? word[j] & 0xffffu : 0xff80u) |
                    (m >> (2 * j + 1) & 1 ? word[j] & 0xffff0000u : 0xff800000u);
      }
    }
    if (v >= begin && v + VN <= end) {
      *reinterpret_cast<uint4*>(y + v) = raw[i];
    } else {
#pragma unroll
      for (int j = 0; j < VN; ++j)
        if (v + j >= begin && v + j < end) y[v + j] = e[j];
    }
  }
  if (a.bias_count) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < BIAS; ++k)
      if (put[k]) Elem<T>::store(y + bt[tid + k * kLogitsThreads], bz[k]);
  }
}

template <typename T, int PER>
static int launch_adjust(const logkv_logits_args_t& a, cudaStream_t st) {
  constexpr int VN = 16 / (int)sizeof(T), SLICE = kLogitsThreads * PER * VN;
  const size_t smem = (a.history ? (size_t)SLICE * 4 : 0) + (size_t)a.bias_count * 8;
  // A row whose start is not aligned reaches VN - 1 tokens further.
  const unsigned slices = (unsigned)(((long long)a.vocab + VN - 1 + SLICE - 1) / SLICE);
  launch_pdl(adjust_logits_kernel<T, PER>, dim3(slices, a.rows), kLogitsThreads, smem, st, a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? LOGKV_OK : (int)e;
}

template <typename T>
static int launch_adjust(const logkv_logits_args_t& a, cudaStream_t st) {
  constexpr int VN = 16 / (int)sizeof(T);
  const long long vectors = (long long)a.rows * ((a.vocab + VN - 1) / VN);
  const long long ctas = vectors / kLogitsThreads;   // with one vector per thread
  if (ctas >= 4 * 148 * 8) return launch_adjust<T, 4>(a, st);
  if (ctas >= 2 * 148 * 4) return launch_adjust<T, 2>(a, st);
  return launch_adjust<T, 1>(a, st);
}

}  // namespace logkv

using namespace logkv;

extern "C" LOGKV_API int logkv_adjust_logits(const logkv_logits_args_t* args, void* stream) {
  if (!args) return LOGKV_E_POINTER;
  logkv_logits_args_t a = *args;
  if (a.dtype != LOGKV_DTYPE_F32 && a.dtype != LOGKV_DTYPE_BF16) return LOGKV_E_DTYPE;
  if (a.rows < 1 || a.rows > 65535 || a.width < 1 || a.vocab < 1 || a.vocab > (1 << 30) || a.history_len < 0 ||
      a.bias_count < 0 || a.bias_count > LOGKV_LOGITS_MAX_BIAS)
    return LOGKV_E_SHAPE;
  auto at = [](const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  const uintptr_t e = a.dtype == LOGKV_DTYPE_F32 ? 4 : 2;
  if (!a.logits || !a.out || !at(a.logits, e) || !at(a.out, e) || !at(a.history, a.history_wide ? 8 : 4) ||
      !at(a.lengths, a.lengths_wide ? 8 : 4) || !at(a.prompts, a.prompts_wide ? 8 : 4) || !at(a.repetitions, 4) ||
      !at(a.presences, 4) || !at(a.frequencies, 4) || !at(a.bias_tokens, a.bias_wide ? 8 : 4) || !at(a.bias_values, 4) ||
      !at(a.mask, 4))
    return LOGKV_E_POINTER;
  if (!a.bias_tokens || !a.bias_values) a.bias_count = 0;
  if (a.history_len == 0) a.history = nullptr;
  if (!a.repetitions && !(a.repetition > 0.f)) return LOGKV_E_SHAPE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return a.dtype == LOGKV_DTYPE_F32 ? launch_adjust<float>(a, st) : launch_adjust<__nv_bfloat16>(a, st);
}
