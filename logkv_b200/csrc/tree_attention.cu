// Attention of a tree of drafted tokens over the LogKV cache (C ABI in include/logkv_attention.h).
//
// The query rows of a (b, g) lane are its rf heads times T tokens, r = h * T + t.  They attend over
// three segments of keys: the packed prefix (log-mass term), the window, the T drafted tokens under
// the tree's ancestor mask.  The keys of a lane are split over CTAs; every CTA keeps the running
// maximum and sum of its rows' softmax in float32 and leaves (m, l, O) per row, which
// tree_combine_kernel joins in split order.
//
// Bound by HBM (keys and values are read once per 128 query rows) from a few MB per SM on; below that
// by latency.  Measured on B200, device time: 7 drafts of one sequence over 7.8K slots x 8 groups (32 MB)
// 14.8 us; 8 x 26 drafts (260 MB) 53 us, 0.76 of the measured copy bandwidth; 32 x 64 drafts (1.06 GB,
// 131 GFLOP) 176-212 us, 0.77-0.93.
#include <algorithm>
#include <cstring>

#include "attn_common.cuh"

namespace logkv {

constexpr int32_t kStatusBadParent = 1 << 18;
constexpr int kTreeMaxTokens = LOGKV_TREE_MAX_TOKENS;
constexpr int kTreeWords = kTreeMaxTokens / 32;

struct TreeGeo {
  int B, G, H, rf, T, D;
  int rcap, rcount;
  int nsplit;   // splits of the grid; a lane uses tree_splits() of them
  int nsmin;    // splits that fill the SMs
  int upw;      // key tiles a split has at least (a tile per warp)
  float scale_log2, mass_log2;   // score = dot * scale_log2 + mass * mass_log2, in the log2 domain
  const void* q;
  const void* kn;
  const void* vn;
  long long qs[3], ks[3], vs[3];
  const void* parents;
  long long pstride;
  int wide;
};

// Splits of a lane with `units` key tiles (the same value in the attention kernel and the combine).
__device__ __forceinline__ int tree_splits(const TreeGeo& a, int units) {
  return max(1, min(a.nsplit, min(a.nsmin, units / a.upw)));
}

__device__ __forceinline__ int prefix_length(const logkv_prefix_t& pre, int ln) {
  return min(max(pre.length[ln], 0), pre.capacity);
}

// Ancestor masks of batch row b: bit j of mask[t] = token t sees token j; 0 for an absent token.
// Pointer jumping without rounds: up[t] is the next token of t's chain that its mask does not cover
// yet (-1: the committed tokens, -2: an absent token).  A step joins that token's mask and takes over
// its `up`; reading `up` before the mask, and writing the mask before `up`, leaves no gap whatever the
// other tokens' threads have done by then, and a chain ends after about log2 of its length steps.
// Called by `threads` threads, tid in [0, threads), with their barrier, after tree_parents by the same
// threads has landed.
struct TreeSmem {
  uint32_t mask[kTreeMaxTokens][kTreeWords];
  int up[kTreeMaxTokens];
  long long raw[kTreeMaxTokens];   // parents as given (int32 ones packed)
};

// Batch row b's parents into `m.raw` by cp.async, asked for at a kernel's start: under a full memory
// system they take microseconds to come.
__device__ __forceinline__ void tree_parents(const TreeGeo& a, int b, TreeSmem& m, int tid, int threads) {
  for (int t = tid; t < a.T; t += threads) {
    const size_t at = (size_t)b * a.pstride + t;
    if (a.wide) cp_async8(&m.raw[t], static_cast<const long long*>(a.parents) + at);
    else cp_async4(reinterpret_cast<int*>(m.raw) + t, static_cast<const int*>(a.parents) + at);
  }
}

template <typename Sync>
__device__ __forceinline__ void tree_masks(const TreeGeo& a, TreeSmem& m, int32_t* status, int tid, int threads,
                                           Sync sync) {
  const int T = a.T, words = (T + 31) >> 5;
  uint32_t(*mask)[kTreeWords] = m.mask;
  int* up = m.up;
  for (int t = tid; t < T; t += threads) {
    const long long p = a.wide ? m.raw[t] : (long long)reinterpret_cast<const int*>(m.raw)[t];
    const bool bad = p < -2 || p >= t;
    if (bad) set_status(status, kStatusBadParent);
    up[t] = bad ? -2 : (int)p;
    for (int w = 0; w < words; ++w) mask[t][w] = (t >> 5) == w ? 1u << (t & 31) : 0u;
  }
  sync();
  volatile int* vup = up;
  for (int t = tid; t < T; t += threads) {
    volatile uint32_t* mine = mask[t];
    int u = up[t];
    while (u >= 0) {   // u falls with every step
      const int next = vup[u];
      __threadfence_block();
      volatile uint32_t* theirs = mask[u];
      for (int w = 0; w <= u >> 5; ++w) mine[w] = mine[w] | theirs[w];
      __threadfence_block();
      vup[t] = next;
      u = next;
    }
  }
  sync();
  for (int t = tid; t < T; t += threads)
    if (up[t] == -2)
      for (int w = 0; w < words; ++w) mask[t][w] = 0u;
  sync();
}

__device__ __forceinline__ bool tree_absent(const uint32_t (*mask)[kTreeWords], int t) {
  return !(mask[t][t >> 5] >> (t & 31) & 1);   // a token that is there sees itself
}

// Partial of one row and split: [m, l, -, -, O[D]], O relative to 2^m; l = -1 marks a row of an absent
// token (written by the splits that hold drafted tokens).
__device__ __forceinline__ float* tree_part(float* part, const TreeGeo& a, int split, size_t row) {
  return part + ((size_t)split * a.B * a.H * a.T + row) * (a.D + 4);
}

// ---------------------------------------------------------------- bf16: mma.sync, 16 query rows per CTA
// The 16 rows are the M of mma.sync.m16n8k16.  Each of the 4 warps streams 16-slot tiles of its own
// through a private ring of cp.async stages (XOR-swizzled for ldmatrix); tiles do not cross segments.
// Used up to 16 rows (tree_tc below has the measurements), and in tiles of 16 rows for the head dims that the
// tcgen05 kernel has no shape for.
constexpr int kTreeWarps = 4;
constexpr int kTreeStages = 3;

// The four warps' results of a CTA's 16 rows, joined in warp order: the split's partial, or the output
// where a lane has one split.  `ring`: each warp's own shared memory, ring_bytes apart.
template <typename T, int D, int DT>
__device__ __forceinline__ void tree_join_warps(const TreeGeo& a, unsigned char* ring, size_t ring_bytes,
                                                float (*wm_)[16], float (*wl_)[16], float (&o)[DT][4], float m0,
                                                float m1, float l0, float l1, int ln, int split, int row0, int NQ,
                                                bool drafts, const TreeSmem& tree, T* out, float* part) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, t4 = lane & 3, T_ = a.T;
  unsigned char* wbase = ring + warp * ring_bytes;
  float* wacc = reinterpret_cast<float*>(wbase);
  if (t4 == 0) {
    wm_[warp][g8] = m0;
    wl_[warp][g8] = l0;
    wm_[warp][g8 + 8] = m1;
    wl_[warp][g8 + 8] = l1;
  }
#pragma unroll
  for (int jd = 0; jd < DT; ++jd) {
    const int c0 = jd * 8 + 2 * t4;
    *reinterpret_cast<float2*>(wacc + g8 * D + c0) = make_float2(o[jd][0], o[jd][1]);
    *reinterpret_cast<float2*>(wacc + (g8 + 8) * D + c0) = make_float2(o[jd][2], o[jd][3]);
  }
  __syncthreads();
  const size_t orow = (size_t)ln * a.rf * T_ + row0;
  const bool whole = a.nsplit == 1;   // no partials, no combine
  if (tid < NQ) {
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < kTreeWarps; ++w) mx = fmaxf(mx, wm_[w][tid]);
    float l = 0.f, f[kTreeWarps];
#pragma unroll
    for (int w = 0; w < kTreeWarps; ++w) {
      f[w] = wm_[w][tid] == -INFINITY ? 0.f : exp2f(wm_[w][tid] - mx);
      l += wl_[w][tid] * f[w];
    }
    const bool absent = drafts && tree_absent(tree.mask, (row0 + tid) % T_);
#pragma unroll
    for (int w = 0; w < kTreeWarps; ++w) wm_[w][tid] = whole ? f[w] / l : f[w];
    wl_[0][tid] = absent ? 1.f : 0.f;
    if (!whole) *reinterpret_cast<float2*>(tree_part(part, a, split, orow + tid)) = make_float2(mx, absent ? -1.f : l);
  }
  __syncthreads();
  for (int x = tid; x < NQ * (D / 4); x += blockDim.x) {
    const int r = x / (D / 4), c = x % (D / 4) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (!whole || wl_[0][r] == 0.f) {
#pragma unroll
      for (int w = 0; w < kTreeWarps; ++w) {
        const float4 y = *reinterpret_cast<const float4*>(ring + w * ring_bytes + (r * D + c) * 4);
        const float f = wm_[w][r];
        v.x = fmaf(y.x, f, v.x);
        v.y = fmaf(y.y, f, v.y);
        v.z = fmaf(y.z, f, v.z);
        v.w = fmaf(y.w, f, v.w);
      }
    }
    if (whole) {
      if constexpr (sizeof(T) == 2)
        *reinterpret_cast<uint2*>(out + (orow + r) * D + c) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
      else
        *reinterpret_cast<float4*>(out + (orow + r) * D + c) = v;
    } else {
      *reinterpret_cast<float4*>(tree_part(part, a, split, orow + r) + 4 + c) = v;
    }
  }
}

template <int D>
struct TreeShape {
  static constexpr int TS = 16, CPR = D / 8, KS = D / 16, DT = D / 8;
  static constexpr int STAGE_BYTES = 2 * TS * D * 2 + TS * 4;   // K, V, mass
  static constexpr size_t smem = (size_t)kTreeWarps * kTreeStages * STAGE_BYTES;
  __device__ __forceinline__ static int swz(int r, int c) {
    if (CPR >= 8) return c ^ (r & 7);
    return c ^ ((r * CPR / 8) & (CPR - 1));
  }
};

template <int D>
__global__ void __launch_bounds__(kTreeWarps * 32, D <= 128 ? 2 : 1)
    tree_mma_kernel(TreeGeo a, logkv_prefix_t pre, const __nv_bfloat16* rk, const __nv_bfloat16* rv,
                    __nv_bfloat16* out, float* part, int32_t* status) {
  using S = TreeShape<D>;
  using B16 = __nv_bfloat16;
  constexpr int TS = S::TS, CPR = S::CPR, KS = S::KS, DT = S::DT, ST = kTreeStages;
  extern __shared__ uint4 smem4[];
  __shared__ TreeSmem tree;
  __shared__ float wm_[kTreeWarps][16], wl_[kTreeWarps][16];
  pdl_entry();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const int g8 = lane >> 2, t4 = lane & 3;
  const int ln = blockIdx.x, split = blockIdx.y, row0 = blockIdx.z * 16, g = ln % a.G, b = ln / a.G;
  const int NQ = min(16, a.rf * a.T - row0), T = a.T;
  tree_parents(a, b, tree, tid, kTreeWarps * 32);
  cp_async_commit();
  const int Lp = prefix_length(pre, ln), R = a.rcount;
  int tok[2];   // tokens of the lane's rows g8 and g8 + 8
  unsigned qa[KS][4];
#pragma unroll
  for (int hr = 0; hr < 2; ++hr) {
    const int r = g8 + 8 * hr, row = row0 + min(r, NQ - 1);
    tok[hr] = row % T;
    const B16* qp = static_cast<const B16*>(a.q) + b * a.qs[0] + (g * a.rf + row / T) * a.qs[1] + tok[hr] * a.qs[2];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qa[ks][hr] = r < NQ ? *reinterpret_cast<const unsigned*>(qp + ks * 16 + 2 * t4) : 0u;
      qa[ks][2 + hr] = r < NQ ? *reinterpret_cast<const unsigned*>(qp + ks * 16 + 2 * t4 + 8) : 0u;
    }
  }
  const int up = (Lp + TS - 1) / TS, ur = (R + TS - 1) / TS, uc = (T + TS - 1) / TS, U = up + ur + uc;
  const int ns = tree_splits(a, U);
  if (split >= ns) {
    cp_async_wait<0>();
    return;
  }
  const int u0 = (int)((long long)U * split / ns), u1 = (int)((long long)U * (split + 1) / ns);
  const int mine = (u1 - u0) > warp ? (u1 - u0 - warp + kTreeWarps - 1) / kTreeWarps : 0;
  unsigned char* wbase = reinterpret_cast<unsigned char*>(smem4) + (size_t)warp * ST * S::STAGE_BYTES;
  const unsigned wbase_s = (unsigned)__cvta_generic_to_shared(wbase);
  const B16* kn = static_cast<const B16*>(a.kn) + b * a.ks[0] + g * a.ks[1];
  const B16* vn = static_cast<const B16*>(a.vn) + b * a.vs[0] + g * a.vs[1];

  // Tile u: its segment, first row and row count.
  auto tile = [&](int u, int& first, int& rows) {
    if (u < up) {
      first = u * TS;
      rows = min(TS, Lp - first);
      return 0;
    }
    if (u < up + ur) {
      first = (u - up) * TS;
      rows = min(TS, R - first);
      return 1;
    }
    first = (u - up - ur) * TS;
    rows = min(TS, T - first);
    return 2;
  };
  auto issue = [&](int k, int stage) {
    if (k < mine) {
      int first, rows;
      const int cls = tile(u0 + warp + k * kTreeWarps, first, rows);
      const size_t r0 = cls == 0 ? (size_t)ln * pre.capacity + first : (size_t)ln * a.rcap + first;
      const B16* kb = cls == 0 ? static_cast<const B16*>(pre.k) + r0 * D : cls == 1 ? rk + r0 * D : kn + first * a.ks[2];
      const B16* vb = cls == 0 ? static_cast<const B16*>(pre.v) + r0 * D : cls == 1 ? rv + r0 * D : vn + first * a.vs[2];
      const long long kst = cls == 2 ? a.ks[2] : D, vst = cls == 2 ? a.vs[2] : D;
      unsigned char* sk = wbase + (size_t)stage * S::STAGE_BYTES;
      unsigned char* sv = sk + TS * D * 2;
      float* sm = reinterpret_cast<float*>(sk + 2 * TS * D * 2);
#pragma unroll
      for (int i = 0; i < (TS * CPR + 31) / 32; ++i) {
        const int flat = i * 32 + lane, r = flat / CPR, c = flat % CPR;
        if (flat < TS * CPR) {
          const int off = r * D * 2 + S::swz(r, c) * 16;
          if (r < rows) {
            cp_async16(sk + off, kb + r * kst + c * 8);
            cp_async16(sv + off, vb + r * vst + c * 8);
          } else {
            *reinterpret_cast<uint4*>(sk + off) = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(sv + off) = make_uint4(0, 0, 0, 0);
          }
        }
      }
      if (lane < TS) {
        if (cls == 0 && lane < rows) cp_async4(sm + lane, pre.mass + r0 + lane);
        else sm[lane] = 0.f;
      }
    }
    cp_async_commit();
  };

  float o[DT][4];
#pragma unroll
  for (int j = 0; j < DT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
#pragma unroll
  for (int k = 0; k < ST - 1; ++k) issue(k, k);
  if (u1 > up + ur) {   // uniform over the block; the parents' copies are the oldest group
    cp_async_wait<ST - 1>();
    tree_masks(a, tree, status, tid, kTreeWarps * 32, [] { __syncthreads(); });
  }
  for (int k = 0; k < mine; ++k) {
    issue(k + ST - 1, (k + ST - 1) % ST);
    cp_async_wait<ST - 1>();
    __syncwarp();
    const int stage = k % ST;
    int first, rows;
    const int cls = tile(u0 + warp + k * kTreeWarps, first, rows);
    unsigned char* st = wbase + (size_t)stage * S::STAGE_BYTES;
    const unsigned sk = wbase_s + stage * S::STAGE_BYTES, sv = sk + TS * D * 2;
    const float* sm = reinterpret_cast<const float*>(st + 2 * TS * D * 2);
    // Columns each row sees; drafted tokens whose V is not finite, taken out of the product below.
    unsigned see0 = (1u << rows) - 1, see1 = see0, poison = 0;
    if (cls == 2) {
      see0 = tree.mask[tok[0]][first >> 5] >> (first & 31) & see0;
      see1 = tree.mask[tok[1]][first >> 5] >> (first & 31) & see1;
      unsigned char* v = st + TS * D * 2;
      const int r = lane & 15;   // two lanes per row of V
      bool bad = false;
      for (int c = lane >> 4; c < CPR; c += 2) {
        uint4 x = *reinterpret_cast<const uint4*>(v + r * D * 2 + c * 16);
        unsigned* w = reinterpret_cast<unsigned*>(&x);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool lo = (w[i] & 0x7f80u) == 0x7f80u, hi = (w[i] & 0x7f800000u) == 0x7f800000u;
          bad |= lo | hi;
          w[i] &= (lo ? 0xffff0000u : ~0u) & (hi ? 0xffffu : ~0u);
        }
        *reinterpret_cast<uint4*>(v + r * D * 2 + c * 16) = x;
      }
      poison = __ballot_sync(0xffffffffu, bad);
      poison = (poison | poison >> 16) & 0xffffu;
      __syncwarp();
    }
    float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int mi = lane >> 3, rr = (mi >> 1) * 8 + (lane & 7), cc = 2 * ks + (mi & 1);
      unsigned b0, b1, b2, b3;
      ldsm_x4(sk + rr * D * 2 + S::swz(rr, cc) * 16, b0, b1, b2, b3);
      mma_bf16(sc[0], qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], b0, b1);
      mma_bf16(sc[1], qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], b2, b3);
    }
    float mt0 = -INFINITY, mt1 = -INFINITY;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = 8 * j + 2 * t4 + e;
        const float mass = sm[col] * a.mass_log2;
        sc[j][e] = see0 >> col & 1 ? fmaf(sc[j][e], a.scale_log2, mass) : -INFINITY;
        sc[j][2 + e] = see1 >> col & 1 ? fmaf(sc[j][2 + e], a.scale_log2, mass) : -INFINITY;
        mt0 = fmaxf(mt0, sc[j][e]);
        mt1 = fmaxf(mt1, sc[j][2 + e]);
      }
    }
#pragma unroll
    for (int off = 1; off < 4; off <<= 1) {
      mt0 = fmaxf(mt0, __shfl_xor_sync(0xffffffffu, mt0, off));
      mt1 = fmaxf(mt1, __shfl_xor_sync(0xffffffffu, mt1, off));
    }
    const float mn0 = fmaxf(m0, mt0), mn1 = fmaxf(m1, mt1);
    const float al0 = mn0 == -INFINITY ? 1.f : exp2f(m0 - mn0);
    const float al1 = mn1 == -INFINITY ? 1.f : exp2f(m1 - mn1);
    m0 = mn0;
    m1 = mn1;
    float p[2][4], s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        p[j][e] = sc[j][e] == -INFINITY ? 0.f : exp2f(sc[j][e] - mn0);
        p[j][2 + e] = sc[j][2 + e] == -INFINITY ? 0.f : exp2f(sc[j][2 + e] - mn1);
        s0 += p[j][e];
        s1 += p[j][2 + e];
      }
    }
    if (poison & see0) s0 = NAN;
    if (poison & see1) s1 = NAN;
    l0 = l0 * al0 + s0;
    l1 = l1 * al1 + s1;
    if (__any_sync(0xffffffffu, al0 != 1.f || al1 != 1.f)) {
#pragma unroll
      for (int jd = 0; jd < DT; ++jd) {
        o[jd][0] *= al0;
        o[jd][1] *= al0;
        o[jd][2] *= al1;
        o[jd][3] *= al1;
      }
    }
    // P as bf16 (the matrix instruction's operand type: off by at most 2^-8 relative, as much as
    // the output's own rounding); its row sums l stay float32 sums of the unrounded values.
    const unsigned pa0 = pack_bf16x2(p[0][0], p[0][1]), pa1 = pack_bf16x2(p[0][2], p[0][3]);
    const unsigned pa2 = pack_bf16x2(p[1][0], p[1][1]), pa3 = pack_bf16x2(p[1][2], p[1][3]);
#pragma unroll
    for (int jd = 0; jd < DT; jd += 2) {
      const int mi = lane >> 3, rr = (mi & 1) * 8 + (lane & 7), cc = jd + (mi >> 1);
      unsigned b0, b1, b2, b3;
      ldsm_x4_t(sv + rr * D * 2 + S::swz(rr, cc) * 16, b0, b1, b2, b3);
      mma_bf16(o[jd], pa0, pa1, pa2, pa3, b0, b1);
      mma_bf16(o[jd + 1], pa0, pa1, pa2, pa3, b2, b3);
    }
    __syncwarp();
  }
  cp_async_wait<0>();
  __syncwarp();
#pragma unroll
  for (int off = 1; off < 4; off <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, off);
    l1 += __shfl_xor_sync(0xffffffffu, l1, off);
  }
  tree_join_warps<B16, D, DT>(a, reinterpret_cast<unsigned char*>(smem4), (size_t)ST * S::STAGE_BYTES, wm_, wl_, o, m0, m1,
                              l0, l1, ln, split, row0, NQ, u1 > up + ur, tree, out, part);
}

// ---------------------------------------------------------------- bf16: tcgen05, up to 128 query rows per CTA
// Head dims 64 and 128.  The query rows (padded to the 128 rows of tcgen05.mma.cta_group::1.kind::f16)
// stay in shared memory; the CTA streams its split of the lane's keys in units of 64 slots:
//   warps 0-3  softmax, thread = query row = TMEM lane (warps past the last row leave at once);
//   warp 4     one thread issues S(r) = Q K(r)^T, then O += P(r-1) V(r-1);
//   warp 5     loads K and V: full tiles by TMA (128-byte swizzle, no multicast), a segment's last
//              tile and the drafted tokens' (strided) by cp.async with zero fill.
// Tensor memory, 256 columns: two 64-column score buffers (P as bf16 over the first half of its own
// scores) and O.  K and V have rings of their own: K(r) is free once its scores are done, V(r) once
// its product is; the loader asks in the order in which the tensor core gives them back.  Two CTAs per
// SM cover each other's chain of scores, softmax and product (1.1 us a unit at 128 rows).  Every wait
// is bounded; on expiry a role stops and the status gets bit 17.
constexpr int32_t kStatusTreeTimeout = 1 << 17;
constexpr long long kTreeWaitBudget = 4000000000LL;   // clock cycles (about 2 s)
constexpr int kTreeTcThreads = 192;

template <int D>
struct TreeTcShape {
  static constexpr int TS = kTcTS, ST = D == 128 ? 2 : 4;
  static constexpr int MR = 2 * ST;   // mass stages, at least ST + 2
  static constexpr int Q_BYTES = (D / 64) * 128 * 128, KV_BYTES = (D / 64) * TS * 128;
  static constexpr int OFF_K = Q_BYTES, OFF_V = OFF_K + ST * KV_BYTES, OFF_M = OFF_V + ST * KV_BYTES;
  static constexpr size_t smem = OFF_M + MR * TS * 4 + 1024;   // + alignment slack
  static constexpr uint32_t COLS = 256;
};

// K/V rows of the prefix and the window as tensor maps (64 x 64 boxes).
struct TreeMaps {
  CUtensorMap k[2];
  CUtensorMap v[2];
};

template <int D>
__global__ void __launch_bounds__(kTreeTcThreads, 2)
    tree_tc_kernel(TreeGeo a, logkv_prefix_t pre, const __nv_bfloat16* rk, const __nv_bfloat16* rv, __nv_bfloat16* out,
                   float* part, int32_t* status, const __grid_constant__ TreeMaps maps, int tma_mask, int tile_rows) {
  using S = TreeTcShape<D>;
  using B16 = __nv_bfloat16;
  constexpr int TS = S::TS, ST = S::ST, MR = S::MR, CPR = D / 8;
  extern __shared__ uint4 smem4[];
  __shared__ TreeSmem tree;
  __shared__ uint64_t q_full, k_full[ST], v_full[ST], k_empty[ST], v_empty[ST], m_full[MR], s_full[2], p_full[2],
      pv_done[2];
  __shared__ uint32_t sh_tmem;
  __shared__ uint32_t sh_poison[ST][2];   // drafted tokens of the stage whose V is not finite
  if (threadIdx.x < 4) tc::prefetch_tensormap(threadIdx.x < 2 ? &maps.k[threadIdx.x] : &maps.v[threadIdx.x - 2]);
  pdl_entry();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int ln = blockIdx.x, split = blockIdx.y, g = ln % a.G, b = ln / a.G, T = a.T;
  const int row0 = blockIdx.z * tile_rows, NQ = min(tile_rows, a.rf * T - row0);
  const int Lp = prefix_length(pre, ln), R = a.rcount;
  const int up = (Lp + TS - 1) / TS, ur = (R + TS - 1) / TS, U = up + ur + (T + TS - 1) / TS;
  const int ns = tree_splits(a, U);
  if (split >= ns) return;
  // The drafted tokens' units cost about four more (copied and checked by one warp, masks): the last
  // split gets that many fewer.  pad < U / ns, so no split is empty.
  const int pad = min(4, U / ns - 1), W = U + (ns > 1 ? max(pad, 0) : 0);
  const int u0 = (int)((long long)W * split / ns), n = min(U, (int)((long long)W * (split + 1) / ns)) - u0;
  unsigned char* raw = reinterpret_cast<unsigned char*>(smem4);
  unsigned char* base = raw + ((1024u - (tc::smem_u32(raw) & 1023u)) & 1023u);
  const uint32_t base_s = tc::smem_u32(base);
  const int live = (NQ + 31) / 32;   // softmax warps with rows
  if (tid == 0) {
    tc::mbar_init(&q_full, 32 * live);
    for (int i = 0; i < ST; ++i) {
      tc::mbar_init(&k_full[i], 1);
      tc::mbar_init(&v_full[i], 1);
      tc::mbar_init(&k_empty[i], 1);
      tc::mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < MR; ++i) tc::mbar_init(&m_full[i], 1);
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&s_full[i], 1);
      tc::mbar_init(&p_full[i], 32 * live);
      tc::mbar_init(&pv_done[i], 1);
    }
    tc::mbar_fence_init();
  }
  if (warp == 0) {
    tc::tmem_alloc(&sh_tmem, S::COLS);
    tc::tmem_relinquish();
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = sh_tmem, t_o = tmem + 128u;
  auto t_s = [&](int r) { return tmem + 64u * (r & 1); };
  auto unit = [&](int u, int& first, int& rows) {
    if (u < up) {
      first = u * TS;
      rows = min(TS, Lp - first);
      return 0;
    }
    if (u < up + ur) {
      first = (u - up) * TS;
      rows = min(TS, R - first);
      return 1;
    }
    first = (u - up - ur) * TS;
    rows = min(TS, T - first);
    return 2;
  };
  auto fail = [&]() {
    if (status) atomicOr(status, kStatusTreeTimeout);
  };

  if (warp == 5) {
    // ------------------------------------------------ loader
    auto row_of = [&](int cls, int first) { return cls == 0 ? (size_t)ln * pre.capacity + first : (size_t)ln * a.rcap + first; };
    // Slot j's mass of unit r: read a unit ahead and not touched (so not waited for) until it is stored.
    auto mass_of = [&](int r, int j) {
      int first, rows;
      const int cls = unit(u0 + r, first, rows);
      return cls == 0 && j < rows ? pre.mass[row_of(0, first) + j] : 0.f;
    };
    auto copy_rows = [&](unsigned char* dst, const B16* src, long long stride, int rows) {
      for (int flat = lane; flat < TS * CPR; flat += 32) {
        const int r = flat / CPR, c = flat % CPR;
        unsigned char* d = dst + (c >> 3) * (TS * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
        if (r < rows) cp_async16(d, src + r * stride + c * 8);
        else *reinterpret_cast<uint4*>(d) = make_uint4(0, 0, 0, 0);
      }
      cp_async_commit();
      cp_async_wait<0>();
      __syncwarp();
    };
    auto load = [&](int r, bool is_v) {
      const int st = r % ST;
      uint64_t* empty = is_v ? &v_empty[st] : &k_empty[st];
      uint64_t* full = is_v ? &v_full[st] : &k_full[st];
      if (r >= ST && !__all_sync(0xffffffffu, tc::mbar_wait(empty, (r / ST - 1) & 1, kTreeWaitBudget))) return false;
      int first, rows;
      const int cls = unit(u0 + r, first, rows);
      unsigned char* dst = base + (is_v ? S::OFF_V : S::OFF_K) + st * S::KV_BYTES;
      if (rows == TS && cls < 2 && (tma_mask >> cls & 1)) {
        if (lane == 0) {
          tc::fence_proxy_async();   // earlier plain stores to this stage before the asynchronous ones
          tc::mbar_arrive_expect_tx(full, S::KV_BYTES);
          const CUtensorMap* map = is_v ? &maps.v[cls] : &maps.k[cls];
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
            tc::tma_load_2d(tc::smem_u32(dst) + c * (TS * 128), map, c * 64, (int)row_of(cls, first), full);
        }
        return true;
      }
      const B16* src;
      long long stride = D;
      if (cls == 2) {
        stride = is_v ? a.vs[2] : a.ks[2];
        src = is_v ? static_cast<const B16*>(a.vn) + b * a.vs[0] + g * a.vs[1]
                   : static_cast<const B16*>(a.kn) + b * a.ks[0] + g * a.ks[1];
        src += first * stride;
      } else {
        src = (cls == 0 ? static_cast<const B16*>(is_v ? pre.v : pre.k) : is_v ? rv : rk) + row_of(cls, first) * D;
      }
      copy_rows(dst, src, stride, rows);
      if (is_v && cls == 2) {
        // Drafted tokens whose V is not finite leave the product; the rows that see them get a NaN sum.
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r_ = 32 * h + lane;
          bool bad = false;
          for (int c = 0; c < CPR; ++c) {
            uint4* p = reinterpret_cast<uint4*>(dst + (c >> 3) * (TS * 128) + r_ * 128 + (((c & 7) ^ (r_ & 7)) << 4));
            uint4 x = *p;
            unsigned* w = reinterpret_cast<unsigned*>(&x);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const bool lo = (w[i] & 0x7f80u) == 0x7f80u, hi = (w[i] & 0x7f800000u) == 0x7f800000u;
              bad |= lo | hi;
              w[i] &= (lo ? 0xffff0000u : ~0u) & (hi ? 0xffffu : ~0u);
            }
            *p = x;
          }
          const unsigned m = __ballot_sync(0xffffffffu, bad);
          if (lane == 0) sh_poison[st][h] = m;
        }
      }
      tc::fence_proxy_async();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(full);
      return true;
    };
    // The mass terms have a longer ring: K(r) may be loaded once the scores of unit r - ST are done, so
    // once P of unit r - ST - 2 has been written and its mass terms read.
    float m0 = mass_of(0, lane), m1 = mass_of(0, lane + 32);
    bool ok = true;
    for (int r = 0; ok && r <= n; ++r) {
      if (r < n) {
        ok = load(r, false);
        if (!ok) break;
        float* sm = reinterpret_cast<float*>(base + S::OFF_M) + (r % MR) * TS;
        sm[lane] = m0 * a.mass_log2;
        sm[lane + 32] = m1 * a.mass_log2;
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&m_full[r % MR]);
        if (r + 1 < n) {
          m0 = mass_of(r + 1, lane);
          m1 = mass_of(r + 1, lane + 32);
        }
      }
      if (r > 0) ok = load(r - 1, true);
    }
    if (!ok && lane == 0) fail();
  } else if (warp == 4) {
    // ------------------------------------------------ MMA issuer
    if (lane == 0) {
      constexpr uint32_t idesc_s = tc::f16_idesc(128, TS, 0, 0), idesc_o = tc::f16_idesc(128, D, 0, 1);
      bool ok = tc::mbar_wait(&q_full, 0, kTreeWaitBudget);
      for (int r = 0; ok && r <= n; ++r) {
        if (r < n) {
          const int st = r % ST;
          // Scores r overwrite P(r - 2): its product is done.
          ok = tc::mbar_wait(&k_full[st], (r / ST) & 1, kTreeWaitBudget) &&
               (r < 2 || tc::mbar_wait(&pv_done[r & 1], (r / 2 - 1) & 1, kTreeWaitBudget));
          if (!ok) break;
          tc::fence_proxy_async();
          tc::fence_after();
          const uint32_t kbs = base_s + S::OFF_K + st * S::KV_BYTES;
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            const uint64_t da = tc::sw128_desc(base_s + (ks >> 2) * (128 * 128) + (ks & 3) * 32, 16, 1024);
            const uint64_t db = tc::sw128_desc(kbs + (ks >> 2) * (TS * 128) + (ks & 3) * 32, 16, 1024);
            tc::umma_f16(t_s(r), da, db, idesc_s, ks > 0 ? 1u : 0u);
          }
          tc::umma_commit(&k_empty[st]);
          tc::umma_commit(&s_full[r & 1]);
        }
        if (r >= 1) {
          const int v = r - 1, st = v % ST;
          ok = tc::mbar_wait(&v_full[st], (v / ST) & 1, kTreeWaitBudget) &&
               tc::mbar_wait(&p_full[v & 1], (v / 2) & 1, kTreeWaitBudget);
          if (!ok) break;
          tc::fence_proxy_async();
          tc::fence_after();
          const uint32_t vbs = base_s + S::OFF_V + st * S::KV_BYTES;
#pragma unroll
          for (int ks = 0; ks < TS / 16; ++ks) {
            const uint64_t db = tc::sw128_desc(vbs + ks * 16 * 128, TS * 128, 1024);
            tc::umma_f16_ts(t_o, t_s(v) + ks * 8, db, idesc_o, (v > 0 || ks > 0) ? 1u : 0u);
          }
          tc::umma_commit(&v_empty[st]);
          tc::umma_commit(&pv_done[v & 1]);
        }
      }
      if (!ok) fail();
    }
  } else if (warp < live) {
    // ------------------------------------------------ softmax, row `tid`
    const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
    const bool in = tid < NQ;
    const int row = row0 + min(tid, NQ - 1), t = row % T, hh = row / T;
    {
      const B16* qp = static_cast<const B16*>(a.q) + b * a.qs[0] + (g * a.rf + hh) * a.qs[1] + t * a.qs[2];
#pragma unroll
      for (int c = 0; c < CPR; ++c) {
        unsigned char* d = base + (c >> 3) * (128 * 128) + tid * 128 + (((c & 7) ^ (tid & 7)) << 4);
        if (in) cp_async16(d, qp + c * 8);
        else *reinterpret_cast<uint4*>(d) = make_uint4(0, 0, 0, 0);
      }
      if (u0 + n > up + ur) tree_parents(a, b, tree, tid, 32 * live);
      cp_async_commit();
      cp_async_wait<0>();
      tc::fence_proxy_async();
      tc::mbar_arrive(&q_full);
    }
    // The tree's masks while the first keys are on their way.
    if (u0 + n > up + ur)
      tree_masks(a, tree, status, tid, 32 * live,
                 [&] { asm volatile("bar.sync 1, %0;\n" ::"r"(32 * live) : "memory"); });
    float m_used = -INFINITY, l = 0.f;
    bool ok = true;
    for (int r = 0; r < n; ++r) {
      const int st = r % ST;
      int first, rows;
      const int cls = unit(u0 + r, first, rows);
      ok = __all_sync(0xffffffffu, tc::mbar_wait(&m_full[r % MR], (r / MR) & 1, kTreeWaitBudget) &&
                                       tc::mbar_wait(&s_full[r & 1], (r / 2) & 1, kTreeWaitBudget) &&
                                       (cls < 2 || tc::mbar_wait(&v_full[st], (r / ST) & 1, kTreeWaitBudget)));
      if (!ok) break;
      tc::fence_after();
      const float* sm = reinterpret_cast<const float*>(base + S::OFF_M) + (r % MR) * TS;
      float sv[TS];
      {
        uint32_t r64[64];
        tc::tmem_ld64(t_s(r) + lane_off, r64);
#pragma unroll
        for (int j = 0; j < TS; ++j) sv[j] = __uint_as_float(r64[j]);
      }
      float mt = -INFINITY;
      const uint64_t c2 = tc::f2pack(a.scale_log2, a.scale_log2);
#pragma unroll
      for (int j = 0; j < TS; j += 4) {
        const float4 m4 = *reinterpret_cast<const float4*>(sm + j);
        tc::f2unpack(tc::ffma2(tc::f2pack(sv[j], sv[j + 1]), c2, tc::f2pack(m4.x, m4.y)), sv[j], sv[j + 1]);
        tc::f2unpack(tc::ffma2(tc::f2pack(sv[j + 2], sv[j + 3]), c2, tc::f2pack(m4.z, m4.w)), sv[j + 2], sv[j + 3]);
      }
      float spoil = 0.f;
      if (rows < TS || cls == 2) {
        uint32_t lo = rows >= 32 ? ~0u : (1u << rows) - 1, hi = rows >= 64 ? ~0u : rows > 32 ? (1u << (rows - 32)) - 1 : 0u;
        if (cls == 2) {
          lo &= tree.mask[t][first >> 5];
          hi &= tree.mask[t][(first >> 5) + 1];
          if ((lo & sh_poison[st][0]) | (hi & sh_poison[st][1])) spoil = NAN;
        }
#pragma unroll
        for (int j = 0; j < TS; ++j) sv[j] = (j < 32 ? lo >> (j & 31) : hi >> (j & 31)) & 1 ? sv[j] : -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < TS; j += 4) mt = fmaxf(mt, fmaxf(fmaxf(sv[j], sv[j + 1]), fmaxf(sv[j + 2], sv[j + 3])));
      // The running maximum moves only when a unit exceeds it by more than 2^8 (then O is rescaled).
      float alpha = 1.f;
      if (mt > m_used + 8.f || (m_used == -INFINITY && mt != -INFINITY)) {
        alpha = m_used == -INFINITY ? 0.f : tc::ex2(m_used - mt);
        m_used = mt;
      }
      const float msub = m_used == -INFINITY ? 0.f : m_used;
      const uint64_t nm2 = tc::f2pack(-msub, -msub);
      uint64_t ps2 = tc::f2pack(0.f, 0.f);
      uint32_t pk[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        float x0, x1;
        tc::f2unpack(tc::fadd2(tc::f2pack(sv[2 * j], sv[2 * j + 1]), nm2), x0, x1);
        const float p0 = tc::ex2(x0), p1 = tc::ex2(x1);
        ps2 = tc::fadd2(ps2, tc::f2pack(p0, p1));
        pk[j] = pack_bf16x2(p0, p1);   // the matrix instruction's operand type; l sums the unrounded values
      }
      float ps0, ps1;
      tc::f2unpack(ps2, ps0, ps1);
      l = l * alpha + (ps0 + ps1) + spoil;
      if (r > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
        ok = __all_sync(0xffffffffu, tc::mbar_wait(&pv_done[(r - 1) & 1], ((r - 1) / 2) & 1, kTreeWaitBudget));
        if (!ok) break;
        tc::fence_after();
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += 32) {
          uint32_t r32[32];
          tc::tmem_ld32(t_o + lane_off + c0, r32);
#pragma unroll
          for (int j = 0; j < 32; ++j) r32[j] = __float_as_uint(__uint_as_float(r32[j]) * alpha);
          tc::tmem_st32(t_o + lane_off + c0, r32);
        }
      }
      tc::tmem_st32(t_s(r) + lane_off, pk);
      tc::fence_before();
      tc::mbar_arrive(&p_full[r & 1]);
    }
    if (ok) ok = __all_sync(0xffffffffu, tc::mbar_wait(&pv_done[(n - 1) & 1], ((n - 1) / 2) & 1, kTreeWaitBudget));
    if (!ok) {
      if (lane == 0) fail();
    } else {
      tc::fence_after();
      const size_t orow = (size_t)ln * a.rf * T + row;
      const bool absent = u0 + n > up + ur && tree_absent(tree.mask, t);
      const bool whole = a.nsplit == 1;   // no partials, no combine
      float* pp = tree_part(part, a, split, orow);
      const float inv = 1.f / l;
      if (in && !whole) *reinterpret_cast<float2*>(pp) = make_float2(m_used, absent ? -1.f : l);
#pragma unroll 1
      for (int c0 = 0; c0 < D; c0 += 32) {
        uint32_t r32[32];
        tc::tmem_ld32(t_o + lane_off + c0, r32);
        if (!in) continue;
        if (whole) {
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            uint4 w = make_uint4(0u, 0u, 0u, 0u);
            if (!absent) {
              w.x = pack_bf16x2(__uint_as_float(r32[j]) * inv, __uint_as_float(r32[j + 1]) * inv);
              w.y = pack_bf16x2(__uint_as_float(r32[j + 2]) * inv, __uint_as_float(r32[j + 3]) * inv);
              w.z = pack_bf16x2(__uint_as_float(r32[j + 4]) * inv, __uint_as_float(r32[j + 5]) * inv);
              w.w = pack_bf16x2(__uint_as_float(r32[j + 6]) * inv, __uint_as_float(r32[j + 7]) * inv);
            }
            *reinterpret_cast<uint4*>(out + orow * D + c0 + j) = w;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            *reinterpret_cast<float4*>(pp + 4 + c0 + j) =
                make_float4(__uint_as_float(r32[j]), __uint_as_float(r32[j + 1]), __uint_as_float(r32[j + 2]),
                            __uint_as_float(r32[j + 3]));
        }
      }
    }
  }
  tc::fence_before();
  __syncthreads();
  if (warp == 0) {
    tc::fence_after();
    tc::tmem_dealloc(tmem, S::COLS);
  }
}

// ---------------------------------------------------------------- float32: mma.sync in three tf32 products
// As the bf16 kernel, with mma.sync.m16n8k8 (tf32): every float32 operand is split into a tf32 part and
// the tf32 part of the rest (22 bits together), and a product is hi hi + hi lo + lo hi, summed in
// float32; what is left out is below 2^-21 of it.  (Float32 fused products from shared memory, four rows by
// four keys a thread, were bound by shared-memory reads: 23.7 us against 16.5 for 39 rows over 2.2K keys.)
// K and V rows are padded by 16 bytes, so that the fragments' reads fall into 32 different banks.
template <int D>
struct TreeF32Shape {
  static constexpr int TS = 16, LD = D + 4, KS = D / 8, DT = D / 8, CPR = D / 4;
  static constexpr int ST = D == 64 ? 2 : 3;   // two CTAs per SM up to 64 features, one at 128
  static constexpr int STAGE_BYTES = 2 * TS * LD * 4 + TS * 4;   // K, V, mass
  static constexpr size_t smem = (size_t)kTreeWarps * ST * STAGE_BYTES;
  static constexpr int CTAS = D <= 64 ? 2 : 1;   // per SM
};

__device__ __forceinline__ void mma_tf32(float* c, const unsigned* a, unsigned b0, unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void split_tf32(float x, unsigned& hi, unsigned& lo) {
  asm("cvt.rna.tf32.f32 %0, %1;\n" : "=r"(hi) : "f"(x));
  asm("cvt.rna.tf32.f32 %0, %1;\n" : "=r"(lo) : "f"(x - __uint_as_float(hi)));
}
// The same, not moved out of a loop (Q's parts of 64 features and more would not fit the registers).
__device__ __forceinline__ void split_tf32_here(float x, unsigned& hi, unsigned& lo) {
  asm volatile("cvt.rna.tf32.f32 %0, %1;\n" : "=r"(hi) : "f"(x));
  asm volatile("cvt.rna.tf32.f32 %0, %1;\n" : "=r"(lo) : "f"(x - __uint_as_float(hi)));
}
// c += a b for one n8 tile, the operands split.  The three products start from zero and are added to c by a
// rounded float32 sum: the matrix instruction's own accumulation truncates, which over a long sum is a
// bias (relative error 2e-6 where this has 2.5e-7).
__device__ __forceinline__ void mma_split(float* c, const unsigned* ah, const unsigned* al, float x0, float x1) {
  unsigned h0, l0, h1, l1;
  split_tf32(x0, h0, l0);
  split_tf32(x1, h1, l1);
  float d[4] = {0.f, 0.f, 0.f, 0.f};
  mma_tf32(d, al, h0, h1);
  mma_tf32(d, ah, l0, l1);
  mma_tf32(d, ah, h0, h1);
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] += d[i];
}

template <int D>
__global__ void __launch_bounds__(kTreeWarps * 32, TreeF32Shape<D>::CTAS)
    tree_f32_kernel(TreeGeo a, logkv_prefix_t pre, const float* rk, const float* rv, float* out, float* part,
                    int32_t* status) {
  using S = TreeF32Shape<D>;
  constexpr int TS = S::TS, LD = S::LD, KS = S::KS, DT = S::DT, CPR = S::CPR, ST = S::ST;
  extern __shared__ uint4 smem4[];
  __shared__ TreeSmem tree;
  __shared__ float wm_[kTreeWarps][16], wl_[kTreeWarps][16];
  pdl_entry();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const int g8 = lane >> 2, t4 = lane & 3;
  const int ln = blockIdx.x, split = blockIdx.y, row0 = blockIdx.z * 16, g = ln % a.G, b = ln / a.G;
  const int NQ = min(16, a.rf * a.T - row0), T = a.T;
  tree_parents(a, b, tree, tid, kTreeWarps * 32);
  cp_async_commit();
  const int Lp = prefix_length(pre, ln), R = a.rcount;
  int tok[2];   // tokens of the lane's rows g8 and g8 + 8
  float qf[KS][4];   // A fragments: (g8, t4), (g8 + 8, t4), (g8, t4 + 4), (g8 + 8, t4 + 4)
#pragma unroll
  for (int hr = 0; hr < 2; ++hr) {
    const int r = g8 + 8 * hr, row = row0 + min(r, NQ - 1);
    tok[hr] = row % T;
    const float* qp = static_cast<const float*>(a.q) + b * a.qs[0] + (g * a.rf + row / T) * a.qs[1] + tok[hr] * a.qs[2];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[ks][hr] = r < NQ ? qp[ks * 8 + t4] : 0.f;
      qf[ks][2 + hr] = r < NQ ? qp[ks * 8 + t4 + 4] : 0.f;
    }
  }
  const int up = (Lp + TS - 1) / TS, ur = (R + TS - 1) / TS, uc = (T + TS - 1) / TS, U = up + ur + uc;
  const int ns = tree_splits(a, U);
  if (split >= ns) {
    cp_async_wait<0>();
    return;
  }
  const int u0 = (int)((long long)U * split / ns), u1 = (int)((long long)U * (split + 1) / ns);
  const int mine = (u1 - u0) > warp ? (u1 - u0 - warp + kTreeWarps - 1) / kTreeWarps : 0;
  unsigned char* wbase = reinterpret_cast<unsigned char*>(smem4) + (size_t)warp * ST * S::STAGE_BYTES;
  const float* kn = static_cast<const float*>(a.kn) + b * a.ks[0] + g * a.ks[1];
  const float* vn = static_cast<const float*>(a.vn) + b * a.vs[0] + g * a.vs[1];
  auto tile = [&](int u, int& first, int& rows) {
    if (u < up) {
      first = u * TS;
      rows = min(TS, Lp - first);
      return 0;
    }
    if (u < up + ur) {
      first = (u - up) * TS;
      rows = min(TS, R - first);
      return 1;
    }
    first = (u - up - ur) * TS;
    rows = min(TS, T - first);
    return 2;
  };
  auto issue = [&](int k, int stage) {
    if (k < mine) {
      int first, rows;
      const int cls = tile(u0 + warp + k * kTreeWarps, first, rows);
      const size_t r0 = cls == 0 ? (size_t)ln * pre.capacity + first : (size_t)ln * a.rcap + first;
      const float* kb = cls == 0 ? static_cast<const float*>(pre.k) + r0 * D : cls == 1 ? rk + r0 * D : kn + first * a.ks[2];
      const float* vb = cls == 0 ? static_cast<const float*>(pre.v) + r0 * D : cls == 1 ? rv + r0 * D : vn + first * a.vs[2];
      const long long kst = cls == 2 ? a.ks[2] : D, vst = cls == 2 ? a.vs[2] : D;
      float* sk = reinterpret_cast<float*>(wbase + (size_t)stage * S::STAGE_BYTES);
      float* sv = sk + TS * LD;
      float* sm = sv + TS * LD;
#pragma unroll 8
      for (int flat = lane; flat < TS * CPR; flat += 32) {
        const int r = flat / CPR, c = flat % CPR;
        if (r < rows) {
          cp_async16(sk + r * LD + c * 4, kb + r * kst + c * 4);
          cp_async16(sv + r * LD + c * 4, vb + r * vst + c * 4);
        } else {
          *reinterpret_cast<float4*>(sk + r * LD + c * 4) = make_float4(0.f, 0.f, 0.f, 0.f);
          *reinterpret_cast<float4*>(sv + r * LD + c * 4) = make_float4(0.f, 0.f, 0.f, 0.f);
        }
      }
      if (lane < TS) {
        if (cls == 0 && lane < rows) cp_async4(sm + lane, pre.mass + r0 + lane);
        else sm[lane] = 0.f;
      }
    }
    cp_async_commit();
  };
  float o[DT][4];
#pragma unroll
  for (int j = 0; j < DT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
#pragma unroll
  for (int k = 0; k < ST - 1; ++k) issue(k, k);
  if (u1 > up + ur) {   // uniform over the block; the parents' copies are the oldest group
    cp_async_wait<ST - 1>();
    tree_masks(a, tree, status, tid, kTreeWarps * 32, [] { __syncthreads(); });
  }
  for (int k = 0; k < mine; ++k) {
    issue(k + ST - 1, (k + ST - 1) % ST);
    cp_async_wait<ST - 1>();
    __syncwarp();
    int first, rows;
    const int cls = tile(u0 + warp + k * kTreeWarps, first, rows);
    float* sk = reinterpret_cast<float*>(wbase + (size_t)(k % ST) * S::STAGE_BYTES);
    float* sv = sk + TS * LD;
    const float* sm = sv + TS * LD;
    // Columns each row sees; drafted tokens whose V is not finite, taken out of the product below.
    unsigned see0 = (1u << rows) - 1, see1 = see0, poison = 0;
    if (cls == 2) {
      see0 = tree.mask[tok[0]][first >> 5] >> (first & 31) & see0;
      see1 = tree.mask[tok[1]][first >> 5] >> (first & 31) & see1;
      const int r = lane & 15;   // two lanes per row of V
      bool bad = false;
      for (int c = lane >> 4; c < D; c += 2)
        if (!isfinite(sv[r * LD + c])) {
          sv[r * LD + c] = 0.f;
          bad = true;
        }
      poison = __ballot_sync(0xffffffffu, bad);
      poison = (poison | poison >> 16) & 0xffffu;
      __syncwarp();
    }
    float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      unsigned ah[4], al[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (D > 32) split_tf32_here(qf[ks][i], ah[i], al[i]);
        else split_tf32(qf[ks][i], ah[i], al[i]);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
        mma_split(sc[j], ah, al, sk[(8 * j + g8) * LD + 8 * ks + t4], sk[(8 * j + g8) * LD + 8 * ks + t4 + 4]);
    }
    float mt0 = -INFINITY, mt1 = -INFINITY;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = 8 * j + 2 * t4 + e;
        const float mass = sm[col] * a.mass_log2;
        sc[j][e] = see0 >> col & 1 ? fmaf(sc[j][e], a.scale_log2, mass) : -INFINITY;
        sc[j][2 + e] = see1 >> col & 1 ? fmaf(sc[j][2 + e], a.scale_log2, mass) : -INFINITY;
        mt0 = fmaxf(mt0, sc[j][e]);
        mt1 = fmaxf(mt1, sc[j][2 + e]);
      }
    }
#pragma unroll
    for (int off = 1; off < 4; off <<= 1) {
      mt0 = fmaxf(mt0, __shfl_xor_sync(0xffffffffu, mt0, off));
      mt1 = fmaxf(mt1, __shfl_xor_sync(0xffffffffu, mt1, off));
    }
    const float mn0 = fmaxf(m0, mt0), mn1 = fmaxf(m1, mt1);
    const float al0 = mn0 == -INFINITY ? 1.f : exp2f(m0 - mn0);
    const float al1 = mn1 == -INFINITY ? 1.f : exp2f(m1 - mn1);
    m0 = mn0;
    m1 = mn1;
    float p[2][4], s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        p[j][e] = sc[j][e] == -INFINITY ? 0.f : exp2f(sc[j][e] - mn0);
        p[j][2 + e] = sc[j][2 + e] == -INFINITY ? 0.f : exp2f(sc[j][2 + e] - mn1);
        s0 += p[j][e];
        s1 += p[j][2 + e];
      }
    }
    if (poison & see0) s0 = NAN;
    if (poison & see1) s1 = NAN;
    l0 = l0 * al0 + s0;
    l1 = l1 * al1 + s1;
    if (__any_sync(0xffffffffu, al0 != 1.f || al1 != 1.f)) {
#pragma unroll
      for (int jd = 0; jd < DT; ++jd) {
        o[jd][0] *= al0;
        o[jd][1] *= al0;
        o[jd][2] *= al1;
        o[jd][3] *= al1;
      }
    }
    // O += P V, eight slots at a time: slot 8 j + 2 t4 + e is index t4 + 4 e of the product, which makes the
    // scores' fragment P's.
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      unsigned ph[4], pl[4];
      split_tf32(p[j][0], ph[0], pl[0]);
      split_tf32(p[j][2], ph[1], pl[1]);
      split_tf32(p[j][1], ph[2], pl[2]);
      split_tf32(p[j][3], ph[3], pl[3]);
      const float* vr = sv + (8 * j + 2 * t4) * LD + g8;
#pragma unroll
      for (int jd = 0; jd < DT; ++jd) mma_split(o[jd], ph, pl, vr[8 * jd], vr[LD + 8 * jd]);
    }
    __syncwarp();
  }
  cp_async_wait<0>();
  __syncwarp();
#pragma unroll
  for (int off = 1; off < 4; off <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, off);
    l1 += __shfl_xor_sync(0xffffffffu, l1, off);
  }
  tree_join_warps<float, D, DT>(a, reinterpret_cast<unsigned char*>(smem4), (size_t)ST * S::STAGE_BYTES, wm_, wl_, o, m0,
                                m1, l0, l1, ln, split, row0, NQ, u1 > up + ur, tree, out, part);
}

// ---------------------------------------------------------------- combine
// WPR warps per output row (1 or 4): each joins its share of the splits' partials, 32 at a time (lane s
// holds split s's m and l; the O loads of 4 or 16 splits in flight), then the warps in order.  TS: the key
// tile of the kernel that wrote the partials.  The order of the sums is fixed by the split count.
template <typename T, int D, int TS, int WPR>
__global__ void __launch_bounds__(128) tree_combine_kernel(TreeGeo a, logkv_prefix_t pre, const float* part, T* out) {
  constexpr int PER = (D + 127) / 128, NB = WPR > 1 ? 16 : 4;
  __shared__ float sh[4][2 + D];
  pdl_entry();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp % WPR;
  const size_t row = (size_t)blockIdx.x * (4 / WPR) + warp / WPR;
  if (WPR == 1 && row >= (size_t)a.B * a.H * a.T) return;
  const int ln = (int)(row / ((size_t)a.rf * a.T));
  const int units = (prefix_length(pre, ln) + TS - 1) / TS + (a.rcount + TS - 1) / TS + (a.T + TS - 1) / TS;
  const int ns = tree_splits(a, units);
  const size_t stride = (size_t)a.B * a.H * a.T * (D + 4);
  const float* p0 = part + row * (D + 4);
  float m = -INFINITY, l = 0.f;
  bool absent = false;
  float4 o[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  const int share = (ns + WPR - 1) / WPR, end = min(ns, (sub + 1) * share);
  for (int s0 = sub * share; s0 < end; s0 += 32) {
    const int cnt = min(32, end - s0);
    const float2 ml = lane < cnt ? *reinterpret_cast<const float2*>(p0 + (s0 + lane) * stride) : make_float2(-INFINITY, 0.f);
    float mc = ml.x;
#pragma unroll
    for (int off = 16; off; off >>= 1) mc = fmaxf(mc, __shfl_xor_sync(0xffffffffu, mc, off));
    const float mn = fmaxf(m, mc), al = m == -INFINITY ? 0.f : exp2f(m - mn);
    const float w = ml.x == -INFINITY ? 0.f : exp2f(ml.x - mn);
    absent |= __any_sync(0xffffffffu, ml.y < 0.f);
    float lw = ml.y * w;
#pragma unroll
    for (int off = 16; off; off >>= 1) lw += __shfl_xor_sync(0xffffffffu, lw, off);
    l = l * al + lw;
    m = mn;
#pragma unroll
    for (int k = 0; k < PER; ++k) o[k] = make_float4(o[k].x * al, o[k].y * al, o[k].z * al, o[k].w * al);
    for (int t0 = 0; t0 < cnt; t0 += NB) {
      float4 v[NB][PER];
#pragma unroll
      for (int s = 0; s < NB; ++s)
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const int c = 4 * (lane + 32 * k);
          v[s][k] = t0 + s < cnt && c < D ? *reinterpret_cast<const float4*>(p0 + (s0 + t0 + s) * stride + 4 + c)
                                          : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
      for (int s = 0; s < NB; ++s) {
        const float ws = __shfl_sync(0xffffffffu, w, (t0 + s) & 31);
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          o[k].x = fmaf(v[s][k].x, ws, o[k].x);
          o[k].y = fmaf(v[s][k].y, ws, o[k].y);
          o[k].z = fmaf(v[s][k].z, ws, o[k].z);
          o[k].w = fmaf(v[s][k].w, ws, o[k].w);
        }
      }
    }
  }
  if (WPR > 1) {
    if (lane == 0) {
      sh[warp][0] = m;
      sh[warp][1] = absent ? -1.f : l;
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int c = 4 * (lane + 32 * k);
      if (c < D) {
        float* d = &sh[warp][2 + c];
        d[0] = o[k].x, d[1] = o[k].y, d[2] = o[k].z, d[3] = o[k].w;
      }
    }
    __syncthreads();
    m = -INFINITY;
    for (int w = 0; w < WPR; ++w) {
      m = fmaxf(m, sh[w][0]);
      absent |= sh[w][1] < 0.f;
    }
    for (int d = threadIdx.x; d < D; d += 128) {
      float L = 0.f, x = 0.f;
#pragma unroll
      for (int w = 0; w < WPR; ++w) {
        const float f = sh[w][0] == -INFINITY ? 0.f : exp2f(sh[w][0] - m);
        L += sh[w][1] * f;
        x += sh[w][2 + d] * f;
      }
      Elem<T>::store(out + row * D + d, absent ? 0.f : x / L);
    }
    return;
  }
  const float inv = 1.f / l;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int c = 4 * (lane + 32 * k);
    if (c < D) {
      T* dst = out + row * D + c;
      Elem<T>::store(dst, absent ? 0.f : o[k].x * inv);
      Elem<T>::store(dst + 1, absent ? 0.f : o[k].y * inv);
      Elem<T>::store(dst + 2, absent ? 0.f : o[k].z * inv);
      Elem<T>::store(dst + 3, absent ? 0.f : o[k].w * inv);
    }
  }
}

// ---------------------------------------------------------------- host side
struct TreePlan {
  int tile_rows, ts, nsplit, nsmin, upw;   // query rows per CTA, key tile, splits
  bool tc;
};

// tcgen05 or mma.sync in tiles of 16 rows.  Measured at D 128 in us, tcgen05 against mma.sync:
//                          16 rows          17 rows          96 rows
//   7.8K keys, 64 lanes    50.3 : 50.4      50.5 : 81.4      57.9 : 292
//   7.8K keys, 8 lanes     15.1 : 15.2      15.3 : 18.7      21.5 : 37.1
//   1.2K keys, 64 lanes    17.6 : 16.6      17.6 : 22.5      22.4 : 61.2
//   1.2K keys, 8 lanes     14.0 : 11.9      14.1 : 12.3      18.7 : 16.7
//   100 keys, 8 lanes      14.5 :  9.4      14.6 : 10.9      18.3 : 13.3
// Up to 16 rows both read every key once and mma.sync starts up faster; from 17 on it reads them twice or more.
// On short caches it would still win 2 to 5 us there, but the host knows only the prefix's capacity.
static bool tree_tc(const logkv_layout_t& l, long long rows) {
  return l.dtype == LOGKV_DTYPE_BF16 && (l.dim == 64 || l.dim == 128) && rows > 16;
}

// Splits: as many CTAs over all lanes and row tiles as run at once, at least a key tile per warp each.
static TreePlan tree_plan(const logkv_layout_t& l, int heads, int tokens, int prefix_capacity) {
  TreePlan p;
  const bool f32 = l.dtype == LOGKV_DTYPE_F32;
  const long long rows = (long long)(heads / l.groups) * tokens;
  p.tc = tree_tc(l, rows);
  const int most = p.tc ? 128 : 16;
  const long long tiles = (rows + most - 1) / most;
  p.tile_rows = p.tc ? (int)((rows + tiles - 1) / tiles) : most;
  p.ts = p.tc ? kTcTS : 16;
  p.upw = p.tc ? 2 : kTreeWarps;
  const long long ctas = (long long)l.batch * l.groups * tiles;
  const int units = (prefix_capacity + l.recent_capacity + tokens) / p.ts + 3;
  const int per_sm = (f32 && l.dim > 64) || l.dim > 128 ? 1 : 2;
  p.nsmin = (int)std::max(1LL, 148 * per_sm / ctas);
  p.nsplit = std::max(1, std::min(p.nsmin, units / p.upw));
  return p;
}

static bool tree_dim_ok(const logkv_layout_t& l) {
  return l.dim == 16 || l.dim == 32 || l.dim == 64 || l.dim == 128 || (l.dim == 256 && l.dtype == LOGKV_DTYPE_BF16);
}

static int check_tree(const logkv_layout_t* l, int heads, int tokens) {
  const int rc = check_layout(l);
  if (rc) return rc;
  if (heads < l->groups || heads % l->groups || tokens < 1 || tokens > kTreeMaxTokens || !tree_dim_ok(*l))
    return LOGKV_E_SHAPE;
  // Grid limits: row tiles along z.
  if ((long long)(heads / l->groups) * tokens > 16LL * 65535) return LOGKV_E_SHAPE;
  return LOGKV_OK;
}

// Four warps to a row from 9 splits on, which few lanes have: 14 rows over 7.8K keys take 14.9 us against 17.7
// with one warp on 8 lanes (37 splits) and 11.6 against 24.5 on one lane; over 100 keys, where
// two of the splits hold any, 9.4 against 9.0.  With few splits the extra warps only wait: 64 lanes (4 splits), 14 rows
// 53.7 against 49.7 us, 52 rows 63.3 against 52.0.
template <typename T, int D, int TS>
static void launch_tree_combine(const TreeGeo& a, const logkv_prefix_t& pre, const float* part, void* out,
                                cudaStream_t st) {
  const size_t rows = (size_t)a.B * a.H * a.T;
  T* o = static_cast<T*>(out);
  if (a.nsplit > 8) launch_pdl(tree_combine_kernel<T, D, TS, 4>, dim3((unsigned)rows), 128, 0, st, a, pre, part, o);
  else launch_pdl(tree_combine_kernel<T, D, TS, 1>, dim3((unsigned)((rows + 3) / 4)), 128, 0, st, a, pre, part, o);
}

template <int D>
static int launch_tree_bf16(const TreeGeo& a, const TreePlan& p, const logkv_prefix_t& pre, const logkv_state_t& s,
                            const logkv_tree_args_t& x, float* part, cudaStream_t st) {
  using S = TreeShape<D>;
  using B16 = __nv_bfloat16;
  auto kern = tree_mma_kernel<D>;
  if (const int e = smem_limit_once<tree_mma_kernel<D>>(S::smem)) return e;
  const unsigned tiles = (unsigned)((a.rf * a.T + p.tile_rows - 1) / p.tile_rows);
  launch_pdl(kern, dim3(a.B * a.G, p.nsplit, tiles), kTreeWarps * 32, S::smem, st, a, pre,
             static_cast<const B16*>(s.recent_k), static_cast<const B16*>(s.recent_v), static_cast<B16*>(x.out), part,
             x.status);
  if (p.nsplit > 1) launch_tree_combine<B16, D, 16>(a, pre, part, x.out, st);
  return launch_status();
}

// tcgen05: head dims 64 and 128.
template <int D>
static int launch_tree_tc(const TreeGeo& a, const TreePlan& p, const logkv_prefix_t& pre, const logkv_state_t& s,
                          const logkv_tree_args_t& x, float* part, cudaStream_t st) {
  using S = TreeTcShape<D>;
  using B16 = __nv_bfloat16;
  auto kern = tree_tc_kernel<D>;
  if (const int e = smem_limit_once<tree_tc_kernel<D>>(S::smem)) return e;
  TreeMaps maps;
  memset(&maps, 0, sizeof(maps));
  const size_t lanes = (size_t)a.B * a.G;
  int mask = 0;
  // Rows are 32-bit coordinates; larger buffers take the cp.async path.
  if (lanes * pre.capacity < (1ull << 31) && encode_rows_map(&maps.k[0], pre.k, lanes * pre.capacity, D) &&
      encode_rows_map(&maps.v[0], pre.v, lanes * pre.capacity, D))
    mask |= 1;
  if (lanes * a.rcap < (1ull << 31) && encode_rows_map(&maps.k[1], s.recent_k, lanes * a.rcap, D) &&
      encode_rows_map(&maps.v[1], s.recent_v, lanes * a.rcap, D))
    mask |= 2;
  const unsigned tiles = (unsigned)((a.rf * a.T + p.tile_rows - 1) / p.tile_rows);
  launch_pdl(kern, dim3(a.B * a.G, p.nsplit, tiles), kTreeTcThreads, S::smem, st, a, pre,
             static_cast<const B16*>(s.recent_k), static_cast<const B16*>(s.recent_v), static_cast<B16*>(x.out), part,
             x.status, maps, mask, p.tile_rows);
  if (p.nsplit > 1) launch_tree_combine<B16, D, kTcTS>(a, pre, part, x.out, st);
  return launch_status();
}

template <int D>
static int launch_tree_f32(const TreeGeo& a, const TreePlan& p, const logkv_prefix_t& pre, const logkv_state_t& s,
                           const logkv_tree_args_t& x, float* part, cudaStream_t st) {
  using S = TreeF32Shape<D>;
  auto kern = tree_f32_kernel<D>;
  if (const int e = smem_limit_once<tree_f32_kernel<D>>(S::smem)) return e;
  const unsigned tiles = (unsigned)((a.rf * a.T + p.tile_rows - 1) / p.tile_rows);
  launch_pdl(kern, dim3(a.B * a.G, p.nsplit, tiles), kTreeWarps * 32, S::smem, st, a, pre,
             static_cast<const float*>(s.recent_k), static_cast<const float*>(s.recent_v), static_cast<float*>(x.out),
             part, x.status);
  if (p.nsplit > 1) launch_tree_combine<float, D, 16>(a, pre, part, x.out, st);
  return launch_status();
}

}  // namespace logkv

using namespace logkv;

extern "C" {

LOGKV_API size_t logkv_tree_attention_workspace_bytes(const logkv_layout_t* layout, int32_t heads, int32_t tokens,
                                                      int32_t prefix_capacity) {
  if (check_tree(layout, heads, tokens) || prefix_capacity < 0) return 0;
  const TreePlan p = tree_plan(*layout, heads, tokens, prefix_capacity);
  return (size_t)p.nsplit * layout->batch * heads * tokens * (layout->dim + 4) * sizeof(float);
}

LOGKV_API int logkv_tree_attention(const logkv_layout_t* layout, const logkv_state_t* state,
                                   const logkv_prefix_t* prefix, const logkv_tree_args_t* x, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  if (!layout || !state || !prefix || !x) return LOGKV_E_POINTER;
  const int rc = check_tree(layout, x->heads, x->tokens);
  if (rc) return rc;
  if (x->recent_count < 0 || x->recent_count > layout->recent_capacity || prefix->capacity < 0) return LOGKV_E_SHAPE;
  auto at = [](const void* p, uintptr_t n) { return p && (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  auto a16 = [&](const void* p) { return at(p, 16); };
  if (!a16(x->q) || !a16(x->k_new) || !a16(x->v_new) || !a16(x->out) || !a16(workspace) || !a16(state->recent_k) ||
      !a16(state->recent_v) || !a16(prefix->k) || !a16(prefix->v) || !at(prefix->mass, 4) || !at(prefix->length, 4) ||
      !at(x->parents, x->parents_wide ? 8 : 4))
    return LOGKV_E_POINTER;
  const long long e = (long long)esize_of(layout->dtype);
  TreeGeo a{};
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = x->q_strides[i];
    a.ks[i] = x->k_strides[i];
    a.vs[i] = x->v_strides[i];
    if (a.qs[i] * e % 16 || a.ks[i] * e % 16 || a.vs[i] * e % 16) return LOGKV_E_POINTER;
  }
  if (workspace_bytes < logkv_tree_attention_workspace_bytes(layout, x->heads, x->tokens, prefix->capacity))
    return LOGKV_E_WORKSPACE;
  const TreePlan p = tree_plan(*layout, x->heads, x->tokens, prefix->capacity);
  a.B = layout->batch;
  a.G = layout->groups;
  a.H = x->heads;
  a.rf = a.H / a.G;
  a.T = x->tokens;
  a.D = layout->dim;
  a.rcap = layout->recent_capacity;
  a.rcount = x->recent_count;
  a.nsplit = p.nsplit;
  a.nsmin = p.nsmin;
  a.upw = p.upw;
  a.scale_log2 = x->scale * 1.4426950408889634f;
  a.mass_log2 = x->qx * a.scale_log2;
  a.q = x->q;
  a.kn = x->k_new;
  a.vn = x->v_new;
  a.parents = x->parents;
  a.pstride = x->parents_stride;
  a.wide = x->parents_wide;
  float* part = static_cast<float*>(workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p.tc) {
    if (layout->dim == 64) return launch_tree_tc<64>(a, p, *prefix, *state, *x, part, st);
    return launch_tree_tc<128>(a, p, *prefix, *state, *x, part, st);
  }
  if (layout->dtype == LOGKV_DTYPE_BF16) {
    switch (layout->dim) {
      case 16: return launch_tree_bf16<16>(a, p, *prefix, *state, *x, part, st);
      case 32: return launch_tree_bf16<32>(a, p, *prefix, *state, *x, part, st);
      case 64: return launch_tree_bf16<64>(a, p, *prefix, *state, *x, part, st);
      case 128: return launch_tree_bf16<128>(a, p, *prefix, *state, *x, part, st);
      default: return launch_tree_bf16<256>(a, p, *prefix, *state, *x, part, st);
    }
  }
  switch (layout->dim) {
    case 16: return launch_tree_f32<16>(a, p, *prefix, *state, *x, part, st);
    case 32: return launch_tree_f32<32>(a, p, *prefix, *state, *x, part, st);
    case 64: return launch_tree_f32<64>(a, p, *prefix, *state, *x, part, st);
    default: return launch_tree_f32<128>(a, p, *prefix, *state, *x, part, st);
  }
}

}  // extern "C"
