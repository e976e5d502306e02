// Rotary positions of queries and keys, and rows brought into the cache with the rotation on the way (C ABI in
// include/logkv_rotary.h).
//
// With c, s the table rows of a token's position, out = x c + turn(x) s, where turn takes the two halves (or
// pairs) of the rotated features for a plane each: (a, b) -> (a c - b s, b c + a s).  Every element is read
// once and written once, so HBM bounds long chunks and the launch bounds single tokens.
//
// A thread owns one unit of a token: VN features of the first half with their VN partners, or features behind the
// rotated ones (VN, and from the next 16-byte boundary on VW).  It reads its table entries once and walks over the heads
// of all tensors with them, kBatch heads' loads in flight; the heads are cut into chunks when tokens are few.  kBatch 2,
// 3, 4, 8: 35, 33, 31, 34 us for 8 x 2048 tokens of 8 key and 8 value heads (176 MB, 0.86 of the measured copy
// bandwidth), 30, 27, 16.5, 22.5 us for 4 x 1777 interleaved ones of 24 heads of 64 float32 (95 MB, 0.88).
#include <algorithm>

#include "attn_common.cuh"
#include "../../include/logkv_rotary.h"

namespace logkv {

constexpr int32_t kStatusPosition = 1 << 16;   // as the prefix pack's
constexpr int kRotateThreads = 128;
constexpr int kBatch = 4;

template <int BYTES> struct RawVec;
template <> struct RawVec<16> { using type = uint4; };
template <> struct RawVec<8> { using type = uint2; };
template <> struct RawVec<4> { using type = unsigned; };
template <> struct RawVec<2> { using type = unsigned short; };

// VN elements as one access.
template <typename T, int VN>
struct Unit {
  using Raw = typename RawVec<(int)sizeof(T) * VN>::type;
  union {
    Raw raw;
    T e[VN];
  };
  __device__ __forceinline__ Unit() {}
  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const Raw*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Raw*>(p) = raw; }
};

// VN table entries as float32, in 16-byte accesses where VN entries are longer.
template <typename C, int VN>
__device__ __forceinline__ void table_unit(const C* p, float (&f)[VN]) {
  constexpr int W = 16 / (int)sizeof(C) < VN ? 16 / (int)sizeof(C) : VN;
#pragma unroll
  for (int i = 0; i < VN; i += W) {
    Unit<C, W> u;
    u.load(p + i);
#pragma unroll
    for (int j = 0; j < W; ++j) f[i + j] = Elem<C>::load(&u.e[j]);
  }
}

struct RotateGeo {
  const void* cos;
  const void* sin;
  int table_rows, n;   // positions in the tables, rotated features
  int heads, chunk;    // heads of all parts, heads per thread
  int units;           // units of a token: n / 2 / VN rotated ones, then the others up to `wide`, then those behind
  int wide;            // first feature that is copied in units of VW
};

template <typename T, int VN>
__device__ __forceinline__ void copy_heads(const logkv_rotate_part_t& x, const T* src, T* out, T* raw, int at, int h0,
                                           int h1) {
  for (int h = h0; h < h1; h += kBatch) {
    Unit<T, VN> v[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (h + i < h1) v[i].load(src + (h + i) * x.src_strides[1] + at);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (h + i >= h1) break;
      if (raw) v[i].store(raw + (h + i) * x.raw_strides[1] + at);
      if (x.rotate) v[i].store(out + (h + i) * x.rotated_strides[1] + at);
    }
  }
}

template <typename T, typename C, int VN, int VW>
__global__ void __launch_bounds__(kRotateThreads) rotate_kernel(RotateGeo g, logkv_rotate_args_t a) {
  pdl_entry();
  const long long item = (long long)blockIdx.x * kRotateThreads + threadIdx.x;
  const long long items = (long long)a.batch * a.tokens * g.units;
  if (item >= items) return;
  const int u = (int)(item % g.units);
  const long long row = item / g.units;
  const int t = (int)(row % a.tokens), b = (int)(row / a.tokens);
  long long pos = a.pos0 + t;
  if (a.positions) {
    const long long at = b * a.position_strides[0] + t * a.position_strides[1];
    pos = a.positions_wide ? static_cast<const long long*>(a.positions)[at]
                           : (long long)static_cast<const int32_t*>(a.positions)[at];
  }
  const int half = g.n >> 1, pairs = half / VN;
  const bool turned = u < pairs;
  // First element of the unit and of its partner, as read and as written.
  const int mid = (g.wide - g.n) / VN;
  const int lo = turned ? u * VN : u < pairs + mid ? g.n + (u - pairs) * VN : g.wide + (u - pairs - mid) * VW;
  const int hi = lo + half;
  const int in0 = turned && a.interleaved ? 2 * lo : lo, in1 = turned && a.interleaved ? in0 + VN : hi;
  if (u == 0 && blockIdx.y == 0) {
    if (a.positions_out) a.positions_out[b * a.positions_out_stride + t] = pos;
    if (a.ends_out) a.ends_out[b * a.ends_out_stride + t] = a.ends[b * a.ends_stride + t];
  }
  float c0[VN], s0[VN], c1[VN], s1[VN];
  if (turned) {
    if (pos < 0 || pos >= g.table_rows) {
      if (u == 0 && blockIdx.y == 0) set_status(a.status, kStatusPosition);
      pos = pos < 0 ? 0 : g.table_rows - 1;
    }
    const C* ct = static_cast<const C*>(g.cos) + pos * g.n + lo;
    const C* st = static_cast<const C*>(g.sin) + pos * g.n + lo;
    table_unit<C, VN>(ct, c0);
    table_unit<C, VN>(st, s0);
    table_unit<C, VN>(ct + half, c1);
    table_unit<C, VN>(st + half, s1);
  }
  const int first = blockIdx.y * g.chunk, last = min(g.heads, first + g.chunk);
  int base = 0;
  for (int p = 0; p < a.n_parts; ++p) {
    const logkv_rotate_part_t& x = a.parts[p];
    const int h0 = max(first - base, 0), h1 = min(last - base, x.heads);
    base += x.heads;
    if (h0 >= h1) continue;
    const T* src = static_cast<const T*>(x.src) + b * x.src_strides[0] + t * x.src_strides[2];
    T* out = static_cast<T*>(x.rotated) + (x.rotated ? b * x.rotated_strides[0] + t * x.rotated_strides[2] : 0);
    T* raw = static_cast<T*>(x.raw) + (x.raw ? b * x.raw_strides[0] + t * x.raw_strides[2] : 0);
    if (VN < VW && u >= pairs + mid) {   // (units of one size stay in one loop: their warps do not diverge)
      copy_heads<T, VW>(x, src, out, raw, lo, h0, h1);
      continue;
    }
    const bool rot = turned && x.rotate, mix = rot && a.interleaved;
    const int r0 = rot ? in0 : lo, r1 = rot ? in1 : hi;   // values are copied in place
    for (int h = h0; h < h1; h += kBatch) {
      Unit<T, VN> va[kBatch], vb[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (h + i < h1) {
          const T* s = src + (h + i) * x.src_strides[1];
          va[i].load(s + r0);
          if (turned) vb[i].load(s + r1);
        }
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (h + i >= h1) break;
        if (mix && VN > 1) {   // pairs to halves
          Unit<T, VN> ea, eb;
#pragma unroll
          for (int j = 0; j < VN; ++j) {
            ea.e[j] = 2 * j < VN ? va[i].e[2 * j < VN ? 2 * j : 0] : vb[i].e[2 * j >= VN ? 2 * j - VN : 0];
            eb.e[j] = 2 * j + 1 < VN ? va[i].e[2 * j + 1 < VN ? 2 * j + 1 : 0]
                                     : vb[i].e[2 * j + 1 >= VN ? 2 * j + 1 - VN : 0];
          }
          va[i] = ea;
          vb[i] = eb;
        }
        if (raw) {
          T* d = raw + (h + i) * x.raw_strides[1];
          va[i].store(d + lo);
          if (turned) vb[i].store(d + hi);
        }
        if (!x.rotate) continue;
        T* d = out + (h + i) * x.rotated_strides[1];
        if (turned) {
          Unit<T, VN> ya, yb;
#pragma unroll
          for (int j = 0; j < VN; ++j) {
            const float xa = Elem<T>::load(&va[i].e[j]), xb = Elem<T>::load(&vb[i].e[j]);
            Elem<T>::store(&ya.e[j], __fmaf_rn(xa, c0[j], -__fmul_rn(xb, s0[j])));
            Elem<T>::store(&yb.e[j], __fmaf_rn(xb, c1[j], __fmul_rn(xa, s1[j])));
          }
          ya.store(d + lo);
          yb.store(d + hi);
        } else {
          va[i].store(d + lo);
        }
      }
    }
  }
}

template <typename T, typename C, int VN, int VW>
static int launch_rotate(RotateGeo g, const logkv_rotate_args_t& a, cudaStream_t st) {
  g.wide = (g.n + VW - 1) / VW * VW;
  g.units = g.n / 2 / VN + (g.wide - g.n) / VN + (a.dim - g.wide) / VW;
  const long long items = (long long)a.batch * a.tokens * g.units;
  // Heads per thread: all of them once the tokens alone make 512 threads per SM, fewer before that.  2048 tokens of 24
  // heads of 128 in us: 9.0 with 2048 threads per SM (a head each, its table entries as many bytes as its own), 8.1
  // with 1024, 6.8 with 512, 7.8 with 256.
  const long long want = 148LL * 512;
  const int chunks = (int)std::min<long long>(g.heads, std::max(1LL, want / items));
  g.chunk = (g.heads + chunks - 1) / chunks;
  const long long blocks = (items + kRotateThreads - 1) / kRotateThreads;
  if (blocks > 0x7fffffffLL || g.heads > 65535) return LOGKV_E_SHAPE;
  launch_pdl(rotate_kernel<T, C, VN, VW>, dim3((unsigned)blocks, (g.heads + g.chunk - 1) / g.chunk), kRotateThreads, 0, st,
             g, a);
  return launch_status();
}

// vn: elements of a rotated unit; wide: whether the features behind may go in 16-byte units.
template <typename T, typename C>
static int launch_rotate(const RotateGeo& g, const logkv_rotate_args_t& a, int vn, bool wide, cudaStream_t st) {
  constexpr int W = 16 / (int)sizeof(T);
  if (vn == W) return launch_rotate<T, C, W, W>(g, a, st);
  if constexpr (W == 8)
    if (vn == 4) return wide ? launch_rotate<T, C, 4, W>(g, a, st) : launch_rotate<T, C, 4, 4>(g, a, st);
  if (vn == 2) return wide ? launch_rotate<T, C, 2, W>(g, a, st) : launch_rotate<T, C, 2, 2>(g, a, st);
  return wide ? launch_rotate<T, C, 1, W>(g, a, st) : launch_rotate<T, C, 1, 1>(g, a, st);
}

}  // namespace logkv

using namespace logkv;

extern "C" LOGKV_API int logkv_rotate(const logkv_rope_t* rope, const logkv_rotate_args_t* args, void* stream) {
  if (!rope || !args) return LOGKV_E_POINTER;
  const logkv_rotate_args_t& a = *args;
  if (!dtype_ok(a.dtype) || (rope->rope_n && !dtype_ok(rope->dtype))) return LOGKV_E_DTYPE;
  if (a.batch < 1 || a.tokens < 1 || a.dim < 1 || a.n_parts < 1 || a.n_parts > LOGKV_ROTATE_MAX_PARTS ||
      rope->rope_n < 0 || rope->rope_n > a.dim || (rope->rope_n & 1))
    return LOGKV_E_SHAPE;
  if (rope->rope_n && (!rope->cos || !rope->sin || rope->rows < 1)) return LOGKV_E_POINTER;
  if (a.positions && (reinterpret_cast<uintptr_t>(a.positions) & (a.positions_wide ? 7 : 3))) return LOGKV_E_POINTER;
  if ((reinterpret_cast<uintptr_t>(a.positions_out) & 7) || (a.ends_out && !a.ends)) return LOGKV_E_POINTER;
  const uintptr_t e = esize_of(a.dtype), ce = esize_of(rope->dtype);
  RotateGeo g{rope->cos, rope->sin, rope->rows, rope->rope_n, 0, 0, 0, 0};
  // Elements per access: the longest that rows, strides, halves and tables allow.
  uintptr_t bits = 0, tab = rope->rope_n ? reinterpret_cast<uintptr_t>(rope->cos) | reinterpret_cast<uintptr_t>(rope->sin) : 0;
  for (int p = 0; p < a.n_parts; ++p) {
    const logkv_rotate_part_t& x = a.parts[p];
    if (x.heads < 1 || !x.src || (x.rotate && !x.rotated) || (!x.rotate && (!x.raw || x.rotated))) return LOGKV_E_POINTER;
    g.heads += x.heads;
    bits |= reinterpret_cast<uintptr_t>(x.src) | reinterpret_cast<uintptr_t>(x.rotated) | reinterpret_cast<uintptr_t>(x.raw);
    for (int i = 0; i < 3; ++i) {
      bits |= (uintptr_t)x.src_strides[i] * e;
      if (x.rotated) bits |= (uintptr_t)x.rotated_strides[i] * e;
      if (x.raw) bits |= (uintptr_t)x.raw_strides[i] * e;
    }
  }
  if (bits & (e - 1) || tab & (ce - 1)) return LOGKV_E_POINTER;
  int vn = (int)(16 / e);
  const bool wide = !(bits & 15) && a.dim % vn == 0;
  auto fits = [&](int v) {
    return !(bits & (v * e - 1)) && g.n / 2 % v == 0 && a.dim % v == 0 &&
           !(tab & (std::min<uintptr_t>(16, v * ce) - 1));
  };
  while (vn > 1 && !fits(vn)) vn >>= 1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  using B16 = __nv_bfloat16;
  const bool bt = g.n && rope->dtype == LOGKV_DTYPE_BF16;
  if (a.dtype == LOGKV_DTYPE_BF16)
    return bt ? launch_rotate<B16, B16>(g, a, vn, wide, st) : launch_rotate<B16, float>(g, a, vn, wide, st);
  return bt ? launch_rotate<float, B16>(g, a, vn, wide, st) : launch_rotate<float, float>(g, a, vn, wide, st);
}
