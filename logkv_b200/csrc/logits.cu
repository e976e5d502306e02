// Penalties of repeated tokens, biases and grammar masks on next-token logits (C ABI in include/logkv_logits.h).
//
// Bound by HBM: every logit is read once and written once, the mask's bits are read once; below a few MB by the
// launch and one part's latency.
//
// A CTA takes one part of one row.  Eight warps copy the part under its mask.  Others, beside them, go over the
// row's history: tokens of the part set bits of a bitmap in shared memory, a prefix sum over its words numbers the set
// ones, and a second pass lists and counts them under their numbers.  Lists are as long as the history at most, however
// long the part, so that few CTAs read a history.  At the end the listed tokens are put over the copy, each from its
// logit as it was.  Counts are integers: the scan's order does not show.
//
// Measured on B200, device time: 512 rows of 151936 bf16 logits (323 MB) with histories of 1024, 16 biases and masks
// 58 us, 0.84 of the measured copy bandwidth (55 without the masks, 52 the copy alone); 145 rows of 50021 float32 ones
// (60 MB) with histories of 4097 and 37 biases 14 us, 0.65, 8 the copy alone; 4 rows of 32000 3.9 us.
#include <algorithm>

#include "common.cuh"
#include "../../include/logkv_logits.h"

namespace logkv {

constexpr int kLogitsThreads = 256;   // that copy; LT more go over the history and the biases, where there are any
constexpr int logits_ctas(int lt) { return lt > 256 ? 2 : lt > 128 ? 3 : 4; }   // of an SM, at 40 registers a thread
constexpr unsigned kSeen = 0x80000000u;   // counter bit of a token that the prompt holds

__device__ __forceinline__ long long load_int(const void* p, int wide, long long i) {
  return wide ? static_cast<const long long*>(p)[i] : (long long)static_cast<const int32_t*>(p)[i];
}

// Bits of tokens v .. v + n - 1 (n <= 8) of a row's mask; those of tokens past the vocabulary are of no account.
__device__ __forceinline__ unsigned mask_bits(const int32_t* mask, int v, int n, int vocab) {
  const int w0 = v >> 5, w1 = min(v + n - 1, vocab - 1) >> 5;
  const unsigned lo = (unsigned)mask[w0], hi = w1 != w0 ? (unsigned)mask[w1] : 0u;
  return __funnelshift_r(lo, hi, v & 31);
}

// Whether token v, whose logit is z after the copy under the mask, is a banned one.  The look at the mask is code of
// its own, which hardly any token of a history comes to: inline it took 145 rows of 50021 (history 4097, no mask) from
// 14.6 to 15.3 us, this way to 14.8.
__device__ __noinline__ bool mask_bans(const int32_t* mask, int v) { return !(mask[v >> 5] >> (v & 31) & 1); }
__device__ __forceinline__ bool banned(const int32_t* mask, float z, int v) {
  return z == -INFINITY && mask && mask_bans(mask, v);
}

template <int LT>
__device__ __forceinline__ void list_sync() {
  asm volatile("bar.sync 1, %0;\n" ::"n"(LT) : "memory");
}

// A row's history, kInFlight tokens of a thread at a time: visit(index of the first, l) with the tokens' places in
// the part [begin, end) from v0 on, -1 for others; token k's index is the first's + k LT.
constexpr int kInFlight = 8;
template <int LT, typename Visit>
__device__ __forceinline__ void visit_history(const logkv_logits_args_t& a, int r, int length, int v0, int begin, int end,
                                              int tid, Visit visit) {
  const long long h0 = (long long)r * a.history_stride;
  for (int i0 = tid; i0 < length; i0 += kInFlight * LT) {
    int l[kInFlight];
#pragma unroll
    for (int k = 0; k < kInFlight; ++k) {
      const int i = i0 + k * LT;
      const long long v = i < length ? load_int(a.history, a.history_wide, h0 + i) : -1;
      l[k] = v >= begin && v < end ? (int)v - v0 : -1;
    }
    visit(i0, l);
  }
}

// A part's place in shared memory.
struct LogitsGeo {
  int part;       // tokens of a CTA, a multiple of 32
  int listed;     // distinct history tokens that a part can hold; 0 without a history
};

// -inf in the elements of a vector whose bit is 0: the bits spread to the signs of bytes, which a byte permutation
// copies over its element's bytes (14 instructions for 8 elements; a select per element took the copy from 57 to 73 us
// for 512 rows of 151936).
__device__ __forceinline__ unsigned byte_signs(unsigned x, unsigned selector) {   // 8 + i in a nibble: byte i's sign
  unsigned y;
  asm("prmt.b32 %0, %1, %1, %2;" : "=r"(y) : "r"(x), "r"(selector));
  return y;
}
template <int VN>
__device__ __forceinline__ void mask_vector(uint4& x, unsigned allow) {
  unsigned* word = reinterpret_cast<unsigned*>(&x);
#pragma unroll
  for (int h = 0; h < VN / 4; ++h) {
    const unsigned s = ((allow >> (4 * h) & 15u) * 0x10204080u) & 0x80808080u;   // bit i in the sign of byte i
    if constexpr (VN == 4) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const unsigned m = byte_signs(s, 0x8888u + 0x1111u * k);
        word[k] = (word[k] & m) | (0xff800000u & ~m);
      }
    } else {
      const unsigned m0 = byte_signs(s, 0x9988u), m1 = byte_signs(s, 0xbbaau);
      word[2 * h] = (word[2 * h] & m0) | (0xff80ff80u & ~m0);
      word[2 * h + 1] = (word[2 * h + 1] & m1) | (0xff80ff80u & ~m1);
    }
  }
}

// 16 bytes from byte o (a multiple of the element's size) of two neighbouring aligned vectors on.
__device__ __forceinline__ uint4 across(const uint4& a, const uint4& b, unsigned o) {
  const bool two = o & 8, one = o & 4;
  unsigned w0 = two ? a.z : a.x, w1 = two ? a.w : a.y, w2 = two ? b.x : a.z, w3 = two ? b.y : a.w, w4 = two ? b.z : b.x;
  const unsigned w5 = two ? b.w : b.y;
  w0 = one ? w1 : w0, w1 = one ? w2 : w1, w2 = one ? w3 : w2, w3 = one ? w4 : w3, w4 = one ? w5 : w4;
  const unsigned bits = 8 * (o & 3);
  return make_uint4(__funnelshift_r(w0, w1, bits), __funnelshift_r(w1, w2, bits), __funnelshift_r(w2, w3, bits),
                    __funnelshift_r(w3, w4, bits));
}

// How the rows lie: all of them start at 16 bytes (a vector's bits are then in one byte of the mask); the logits' rows
// start where the output's do; neither (a vector is put together from the two aligned ones that hold it).
enum RowsAt { kAligned, kTogether, kApart };

template <typename T, RowsAt AT, int LT>
__global__ void __launch_bounds__(kLogitsThreads + LT, logits_ctas(LT))
    adjust_logits_kernel(logkv_logits_args_t a, LogitsGeo g) {
  constexpr int VN = 16 / (int)sizeof(T), U = AT == kApart ? 2 : 4;   // vectors of a thread in flight
  extern __shared__ __align__(16) unsigned smem[];
  __shared__ int warp_sums[LT / 32];
  const int entries = (a.bias_count + 3) / 4 * 4, words = g.part / 32;
  int* bt = reinterpret_cast<int*>(smem);                         // [entries] biased tokens, -1: not here, or again
  float* bz = reinterpret_cast<float*>(bt + entries);             // [entries] biases, then adjusted logits
  unsigned* again = reinterpret_cast<unsigned*>(bz + entries);    // [words] bits of tokens with several biases
  unsigned* before = again + (entries ? words : 0);               // [words] bits of the biased tokens; later on
                                                                  // the touched ones in front of a word
  unsigned* touched = before + words;                             // [words] bits of the history's tokens
  int* token = reinterpret_cast<int*>(touched + words);           // [listed] by number, in index order
  unsigned* count = reinterpret_cast<unsigned*>(token + g.listed);   // [listed]
  pdl_entry();
  const int r = blockIdx.y, n = r / a.width, w = r % a.width;
  const T* x = static_cast<const T*>(a.logits) + n * a.n_stride + w * a.w_stride;
  T* y = static_cast<T*>(a.out) + n * a.out_n_stride + w * a.out_w_stride;
  // Parts start where the output's 16-byte vectors do: vector j of this one is tokens v0 + j VN and on.  Those of
  // [first, last) lie in the part as a whole; the tokens in front of and behind them are fewer than VN each.
  const int mis = (int)((reinterpret_cast<uintptr_t>(y) & 15) / sizeof(T));
  const int v0 = blockIdx.x * g.part - mis, begin = max(v0, 0), end = min(a.vocab, v0 + g.part);
  if (begin >= end) return;
  const int32_t* mask = a.mask ? a.mask + r * a.mask_stride : nullptr;
  const float rep = a.repetitions ? a.repetitions[r] : a.repetition;
  const float pres = a.presences ? a.presences[r] : a.presence, freq = a.frequencies ? a.frequencies[r] : a.frequency;
  auto adjust = [&](float z, unsigned c) {
    const unsigned k = c & ~kSeen;
    z = z > 0.f ? __fdiv_rn(z, rep) : z * rep;
    return k ? z - fmaf(freq, (float)k, pres) : z;
  };
  int listed = 0;

  if (threadIdx.x < kLogitsThreads) {
    const int tid = threadIdx.x;
    int first = (begin - v0 + VN - 1) / VN, last = (end - v0) / VN;
    const int skew = (int)((reinterpret_cast<uintptr_t>(x + v0) & 15) / sizeof(T));   // of the logits' vectors
    if (AT == kApart) {   // both aligned vectors inside the row
      first = max(first, (skew - v0 + VN - 1) / VN);
      last = min(last, max(0, a.vocab - VN + skew - v0) / VN);
    }
    const uint8_t* mask8 = reinterpret_cast<const uint8_t*>(mask);
    for (int j0 = first + tid; j0 < last; j0 += U * kLogitsThreads) {
      // All loads first: what is worked out in between makes each wait for the one before (28 -> 38 us for 256 rows).
      uint4 raw[U], next[U];
      unsigned m0[U], m1[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int j = j0 + i * kLogitsThreads, v = v0 + j * VN;
        if (j < last) {
          const uint4* s = reinterpret_cast<const uint4*>(x + (AT == kApart ? v - skew : v));
          raw[i] = AT == kApart ? s[0] : __ldcs(s);
          if (AT == kApart) next[i] = s[1];
          if (mask) {   // a vector's bits lie in two bytes at most
            m0[i] = mask8[v >> 3];
            if (AT != kAligned) m1[i] = mask8[(v + VN - 1) >> 3];
          }
        }
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int j = j0 + i * kLogitsThreads;
        if (j >= last) break;
        if (AT == kApart) raw[i] = across(raw[i], next[i], skew * (int)sizeof(T));
        if (mask) mask_vector<VN>(raw[i], (AT == kAligned ? m0[i] : m0[i] | m1[i] << 8) >> ((v0 + j * VN) & 7));
        *reinterpret_cast<uint4*>(y + v0 + j * VN) = raw[i];
      }
    }
    // A row's ragged ends (the whole of a part without a whole vector), element by element.
    if (tid < 2 * VN) {
      const int edge = first < last ? v0 + first * VN : end, tail = first < last ? v0 + last * VN : end;
      for (int v = tid < VN ? begin + tid : tail + tid - VN, to = tid < VN ? edge : end; v < to; v += VN)
        if (mask && !(mask_bits(mask, v, 1, a.vocab) & 1)) Elem<T>::store(y + v, -INFINITY);
        else y[v] = x[v];
    }
  } else {
    const int tid = threadIdx.x - kLogitsThreads, lane = tid & 31;
    // The thread's first bias entry and its logit, asked for before the history.
    auto bias_token = [&](int i) {
      const long long v = load_int(a.bias_tokens, a.bias_wide, r * a.bias_tokens_stride + i);
      return v >= begin && v < end ? (int)v : -1;
    };
    int v_own = -1;
    float b_own = 0.f, x_own = 0.f;
    if (tid < a.bias_count) {
      v_own = bias_token(tid);
      b_own = a.bias_values[r * a.bias_values_stride + tid];
      if (v_own >= 0) x_own = Elem<T>::load(x + v_own);
    }
    auto number = [&](int l) {   // of the part's touched token l
      return before[l >> 5] + __popc(touched[l >> 5] & ((1u << (l & 31)) - 1));
    };
    for (int i = tid; i < words; i += LT) {
      if (entries) again[i] = before[i] = 0u;
      if (g.listed) touched[i] = 0u;
    }
    for (int i = tid; i < g.listed; i += LT) count[i] = 0u;
    list_sync<LT>();
    for (int i = tid; i < entries; i += LT) {
      const int v = i == tid ? v_own : i < a.bias_count ? bias_token(i) : -1;
      bt[i] = v;
      bz[i] = i == tid ? b_own : i < a.bias_count ? a.bias_values[r * a.bias_values_stride + i] : 0.f;
      if (v < 0) continue;
      const int l = v - v0;
      const unsigned bit = 1u << (l & 31);
      if (atomicOr(&before[l >> 5], bit) & bit) atomicOr(&again[l >> 5], bit);
    }
    if (g.listed) {
      const long long len = a.lengths ? load_int(a.lengths, a.lengths_wide, r) : a.length;
      const int length = (int)max(0LL, min(len, (long long)a.history_len));
      const long long pro = a.prompts ? load_int(a.prompts, a.prompts_wide, r) : a.prompt;
      const int prompt = (int)max(0LL, min(pro, (long long)length));
      visit_history<LT>(a, r, length, v0, begin, end, tid, [&](int, const int(&l)[kInFlight]) {
        unsigned word[kInFlight];   // frequent tokens are set once
#pragma unroll
        for (int k = 0; k < kInFlight; ++k) word[k] = l[k] < 0 ? ~0u : *static_cast<volatile unsigned*>(&touched[l[k] >> 5]);
#pragma unroll
        for (int k = 0; k < kInFlight; ++k)
          if (!(word[k] >> (l[k] & 31) & 1)) atomicOr(&touched[l[k] >> 5], 1u << (l[k] & 31));
      });
      list_sync<LT>();
      const int per = (words + LT - 1) / LT, w0 = min(words, tid * per), w1 = min(words, w0 + per);
      int sum = 0, at;
      for (int i = w0; i < w1; ++i) sum += __popc(touched[i]);
      at = sum;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, at, off);
        if (lane >= off) at += up;
      }
      if (lane == 31) warp_sums[tid >> 5] = at;
      list_sync<LT>();
      at -= sum;
#pragma unroll
      for (int i = 0; i < LT / 32; ++i) at += i < tid >> 5 ? warp_sums[i] : 0;
      for (int i = w0; i < w1; ++i) {
        before[i] = at;
        at += __popc(touched[i]);
      }
      list_sync<LT>();
      visit_history<LT>(a, r, length, v0, begin, end, tid, [&](int i, const int(&l)[kInFlight]) {
        int n[kInFlight];
#pragma unroll
        for (int k = 0; k < kInFlight; ++k) n[k] = l[k] < 0 ? 0 : number(l[k]);
#pragma unroll
        for (int k = 0; k < kInFlight; ++k)
          if (l[k] >= 0) {
            token[n[k]] = v0 + l[k];   // the same from every thread that meets the token
            if (i + k * LT < prompt) atomicOr(&count[n[k]], kSeen);
            else atomicAdd(&count[n[k]], 1u);
          }
      });
    }
    if (a.bias_count) {
      // The thread of a token's first entry works out its value, with the other entries' biases where it has several.
      // In place the copy leaves the logit as it was, but for a masked one, which is -inf in the end either way.
      list_sync<LT>();
      constexpr int PER = LOGKV_LOGITS_MAX_BIAS / LT;
      float z[PER];
      unsigned mine = 0;
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int i = tid + k * LT, v = i < a.bias_count ? bt[i] : -1, l = v - v0;
        bool first = v >= 0;
        z[k] = 0.f;
        if (!first) continue;
        float sum = bz[i];
        if (again[l >> 5] >> (l & 31) & 1) {
          sum = 0.f;
#pragma unroll 4
          for (int j = 0; j < entries; j += 4) {
            const int4 t = *reinterpret_cast<const int4*>(bt + j);
            if (t.x != v && t.y != v && t.z != v && t.w != v) continue;
            const float4 b = *reinterpret_cast<const float4*>(bz + j);
            first &= (t.x != v || j >= i) && (t.y != v || j + 1 >= i) && (t.z != v || j + 2 >= i) &&
                     (t.w != v || j + 3 >= i);
            sum += t.x == v ? b.x : 0.f;
            sum += t.y == v ? b.y : 0.f;
            sum += t.z == v ? b.z : 0.f;
            sum += t.w == v ? b.w : 0.f;
          }
          if (!first) continue;
        }
        mine |= 1u << k;
        z[k] = k == 0 ? x_own : Elem<T>::load(x + v);
        if (g.listed && touched[l >> 5] >> (l & 31) & 1) z[k] = adjust(z[k], count[number(l)]);
        z[k] += sum;
        if (mask && !(mask_bits(mask, v, 1, a.vocab) & 1)) z[k] = -INFINITY;
      }
      list_sync<LT>();
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int i = tid + k * LT;
        if (i >= a.bias_count) break;
        bz[i] = z[k];
        if (!(mine >> k & 1)) bt[i] = -1;
      }
    }
  }
  if (!g.listed && !a.bias_count) return;
  __syncthreads();
  if (g.listed) {
#pragma unroll
    for (int i = 0; i < LT / 32; ++i) listed += warp_sums[i];
    for (int i = threadIdx.x; i < listed; i += kLogitsThreads + LT) {
      T* e = y + token[i];
      const float z = Elem<T>::load(e);
      // The mask has the last word: a banned token stays -inf whatever its penalties are (they may be infinite).
      if (banned(mask, z, token[i])) continue;
      Elem<T>::store(e, adjust(z, count[i]));
    }
  }
  if (a.bias_count) {
    __syncthreads();
    for (int i = threadIdx.x; i < a.bias_count; i += kLogitsThreads + LT)
      if (bt[i] >= 0) Elem<T>::store(y + bt[i], bz[i]);
  }
}

template <typename T, RowsAt AT, int LT>
static int launch_adjust(const logkv_logits_args_t& a, cudaStream_t st) {
  constexpr int VN = 16 / (int)sizeof(T);
  constexpr int kMost = 200 << 10;   // shared memory of a CTA at most
  constexpr auto kern = adjust_logits_kernel<T, AT, LT>;
  const long long span = (long long)a.vocab + VN - 1;   // a row whose start is not aligned reaches VN - 1 tokens further
  auto geo = [&](long long parts) {
    LogitsGeo g;
    const long long least = (long long)kLogitsThreads * VN;   // a vector per thread
    g.part = (int)((std::max(least, (span + parts - 1) / parts) + 255) / 256 * 256);
    g.listed = a.history ? std::min(a.history_len, g.part) : 0;
    return g;
  };
  auto bytes = [&](const LogitsGeo& g) {
    const size_t words = g.part / 32, entries = (a.bias_count + 3) / 4 * 4;
    return 4 * (entries * 2 + (entries ? words : 0) + (entries || g.listed ? words : 0) +
                (g.listed ? words + 2 * (size_t)g.listed : 0));
  };
  // Parts: one wave of CTAs, and up to three where nothing but the copy is to do, or where a part is still 16 times as
  // long as the history that each of a row's CTAs goes over, and of 64 KB, beside which going over a short history or
  // the biases does not show.  512 rows of 151936 bf16 (history 1024): 62.4 us in one wave, 58.5 in three; 145 rows of
  // 50021 float32 (eight list warps): history 4097 18 in one wave, 26 in two, 33 in three; 64 8.7 in one, 13.5 in three; the copy alone
  // 9.7 in one, 7.7 in three.
  const long long wave = 148 * logits_ctas(LT);
  long long room = a.vocab;
  if (a.history || a.bias_count) room = room * (long long)sizeof(T) >> 16;
  if (a.history) room = std::min(room, a.vocab / (16LL * a.history_len));
  LogitsGeo g = geo(std::max({1LL, wave / a.rows, std::min(3 * wave / a.rows, room)}));
  for (long long parts = 2; bytes(g) > kMost; parts *= 2) g = geo(parts);
  if (const int e = smem_limit_once<kern>(kMost)) return e;
  launch_pdl(kern, dim3((unsigned)((span + g.part - 1) / g.part), a.rows),
             kLogitsThreads + (g.listed || a.bias_count ? LT : 0), bytes(g), st, a, g);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? LOGKV_OK : (int)e;
}

// Eight warps for long histories, sixteen where they are long beside the row, too (an SM then holds three and two CTAs
// instead of four).  With 4, 8 and 16: 145 rows of 50021, history 4097 23, 17, 14 us; 512 rows of 151936, history 1024
// 58.5, 64, -, 4097 -, 68, 79, 8192 -, 99, 97, 20000 -, 176, 123.  Sixteen for many biases, too, whose repeats are
// compared entry by entry (1024 with repeats in 60 rows of 88413: 101 us with four, 44 with sixteen).
template <typename T, RowsAt AT>
static int launch_adjust(const logkv_logits_args_t& a, cudaStream_t st) {
  if (a.bias_count > 512) return launch_adjust<T, AT, 512>(a, st);
  if (!a.history || a.history_len <= 2048) return launch_adjust<T, AT, 128>(a, st);
  return a.vocab < 20LL * a.history_len ? launch_adjust<T, AT, 512>(a, st) : launch_adjust<T, AT, 256>(a, st);
}

// One case for all took 256 rows of 151936 masked bf16 logits from 27.6 to 29.4 us where they are aligned; without the
// second and third, rows of 151643 took 39 us (30.6) contiguous and 53 (34.6) padded to 151936.
template <typename T>
static int launch_adjust(const logkv_logits_args_t& a, cudaStream_t st) {
  const uintptr_t e = sizeof(T);
  auto all = [&](uintptr_t base, int64_t w, int64_t n) {   // a multiple of 16 bytes in every row
    return !((base | (a.width > 1 ? (uintptr_t)w * e : 0) | (a.rows > a.width ? (uintptr_t)n * e : 0)) & 15);
  };
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.logits), y = reinterpret_cast<uintptr_t>(a.out);
  if (!all(x - y, a.w_stride - a.out_w_stride, a.n_stride - a.out_n_stride)) return launch_adjust<T, kApart>(a, st);
  return all(y, a.out_w_stride, a.out_n_stride) ? launch_adjust<T, kAligned>(a, st) : launch_adjust<T, kTogether>(a, st);
}

}  // namespace logkv

using namespace logkv;

extern "C" LOGKV_API int logkv_adjust_logits(const logkv_logits_args_t* args, void* stream) {
  if (!args) return LOGKV_E_POINTER;
  logkv_logits_args_t a = *args;
  if (a.dtype != LOGKV_DTYPE_F32 && a.dtype != LOGKV_DTYPE_BF16) return LOGKV_E_DTYPE;
  if (a.rows < 1 || a.rows > 65535 || a.width < 1 || a.vocab < 1 || a.vocab > (1 << 30) || a.history_len < 0 ||
      a.history_len > (1 << 30) || a.bias_count < 0 || a.bias_count > LOGKV_LOGITS_MAX_BIAS)
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
