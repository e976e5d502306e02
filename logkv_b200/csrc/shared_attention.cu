// Attention of batch rows that share a long prefix of the LogKV cache (C ABI in include/logkv_attention.h).
//
// The rows of a request (W beams forked from one row) hold the same packed prefix and the same first window rows.
// Softmax attention over a union of key sets is joined from the parts' maxima m, sums l and products O,
//   m = max m_i,  l = sum l_i 2^(m_i - m),  O = sum O_i 2^(m_i - m),  out = O / l,
// so the shared keys are read once per row tile of a request's W rf T query rows (128 rows on tcgen05, that is bf16 of
// head dim 64 or 128 and more than 16 rows; 16 elsewhere; a "shared lane" is a request and a KV group), and every batch
// row's own keys - the rest of its window and the new tokens - once by its rf T rows (an "own lane").  Both kinds of
// lanes are split over CTAs of one launch, which leave (m, l, O) per row and split; share_combine_kernel joins them in a
// fixed order, the shared splits first.
//
// Bound by HBM from a few MB per SM on: keys and values are read once per 128 (16) query rows.  Measured on B200, device
// time: 8 requests of 8 rows over 7.8K shared and 242 own keys (8 groups, head dim 128, bf16: 314 MB) 61 us, 0.78 of the
// measured copy bandwidth, where log_kv_chunk_attention takes 367; one request of 4 rows (31 MB) 12.6 us (34); below that
// latency: 3 requests of 16 rows over 2.0K keys 15.1 us.  The join's launch is some 3 us of each (0.5 of them its read of
// the prefix's length, which has to wait for the attention kernel with the rest).
#include <algorithm>
#include <cstring>

#include "attn_common.cuh"

namespace logkv {

struct ShareGeo {
  int B, G, H, rf, T, Tk, W, D;
  int rcap, rcount, w0;   // window: capacity, rows, shared rows
  int causal;             // new token j is seen by query tokens t >= j only
  int nsplit;             // splits of a shared lane in the grid; share_splits() of them are used
  int upw;                // key tiles a split has at least
  int nown;               // splits of an own lane
  int own_warps;          // warps to an own lane's split: 4, 2 or 1
  int shared_lanes, own_lanes;
  int slots;              // CTAs that run at once
  float own_work;         // all own lanes' work in keys, what it takes to start them included
  int tiles, tile_rows;   // row tiles of a shared lane (at most 16 or 128 rows each)
  int own_tiles;          // row tiles of an own lane (16 rows each)
  float scale_log2, mass_log2;   // score = dot * scale_log2 + mass * mass_log2, in the log2 domain
  const void* q;
  const void* kn;
  const void* vn;
  long long qs[3], ks[3], vs[3];
};

// Splits of a shared lane with `units` key tiles (the same value in the attention kernel and the combine): the SMs are
// divided between the two kinds of lanes by their work, so that both end together.  64 shared lanes of 8.0K keys beside
// 512 own ones of 242: 129, 81, 60, 61, 74, 66, 68 us with 1, 2, 3, 4, 5, 6, 8 splits; this gives 3.
__device__ __forceinline__ int share_splits(const ShareGeo& a, int units, int tile_keys) {
  const int ctas = a.shared_lanes * a.tiles;
  // In half CTAs, to the nearest split; every operation rounded on its own, so that both kernels get the same.
  const float work = __fmul_rn((float)(units * tile_keys), (float)ctas);
  const int room = (int)__fdiv_rn(__fmul_rn(2.f * a.slots, work), __fadd_rn(work, a.own_work));
  return max(1, min(a.nsplit, min((room + ctas) / (2 * ctas), units / a.upw)));
}

__device__ __forceinline__ int share_prefix_length(const logkv_prefix_t& pre, int ln) {
  return min(max(pre.length[ln], 0), pre.capacity);
}

// A warp's share of the work, the same for the warps that share a split.  Shared lanes' CTAs come first (lane fastest,
// then split, so that unused splits are dispatched last among them), then those of the own lanes.
struct ShareJob {
  bool own;
  int b, g;        // batch row (the request's first for a shared lane) and group
  int split, slot; // slot: index of the partial among the row's
  int row0, NQ;    // query rows of the lane
  int n0, n1;      // keys of the two segments
  size_t r0;       // first key row of segment 0 (packed prefix, or the window's rows behind w0)
  int ns;          // splits of the lane
  int warps, sub;  // warps of the split and which of them this is
};

// GROUPED: own lanes of fewer than four warps.  Code of its own, since what it takes to tell the groups apart costs the
// calls without them 1 to 2 us.
// What it takes but the prefix's length: all that a kernel may work out before its predecessor has ended.
template <bool GROUPED>
__device__ __forceinline__ ShareJob share_job(const ShareGeo& a, const logkv_prefix_t& pre) {
  ShareJob j;
  int x = blockIdx.x;
  const int shared = a.shared_lanes * a.nsplit * a.tiles, warp = threadIdx.x >> 5;
  j.own = x >= shared;
  if (j.own) {
    j.warps = GROUPED ? a.own_warps : 4;
    j.sub = warp % j.warps;
    x = (x - shared) * (4 / j.warps) + warp / j.warps;
    const int lane = x % a.own_lanes;
    x /= a.own_lanes;
    j.split = x % a.nown;
    j.slot = a.nsplit + j.split;
    j.b = lane / a.G;
    j.g = lane % a.G;
    j.row0 = x / a.nown * 16;
    j.NQ = min(16, a.rf * a.T - j.row0);   // the last CTA's warps past the lanes: 0 or less
    j.n0 = a.rcount - a.w0;
    j.n1 = a.Tk;
    j.r0 = ((size_t)j.b * a.G + j.g) * a.rcap + a.w0;
    j.ns = a.nown;
  } else {
    j.warps = 4;
    j.sub = warp;
    const int lane = x % a.shared_lanes;
    x /= a.shared_lanes;
    j.split = j.slot = x % a.nsplit;
    j.b = lane / a.G * a.W;
    j.g = lane % a.G;
    j.row0 = x / a.nsplit * a.tile_rows;
    j.NQ = min(a.tile_rows, a.W * a.rf * a.T - j.row0);
    j.n0 = 0;
    j.n1 = a.w0;
    j.r0 = ((size_t)j.b * a.G + j.g) * pre.capacity;
    j.ns = 0;
  }
  return j;
}
// The rest: a shared lane's keys and splits.
__device__ __forceinline__ void share_keys(const ShareGeo& a, const logkv_prefix_t& pre, int tile_keys, ShareJob& j) {
  if (j.own) return;
  j.n0 = share_prefix_length(pre, j.b * a.G + j.g);
  j.ns = share_splits(a, (j.n0 + tile_keys - 1) / tile_keys + (j.n1 + tile_keys - 1) / tile_keys, tile_keys);
}

// Key tiles of the split that the warp takes: first, first + warps, ...
struct ShareTiles {
  int un, first, n;   // tiles of segment 0; the warp's
  __device__ __forceinline__ ShareTiles(const ShareJob& j, int ts) {
    un = (j.n0 + ts - 1) / ts;
    const int U = un + (j.n1 + ts - 1) / ts, per = U / j.ns, more = U - per * j.ns;   // the first `more` take one more
    const int u0 = per * j.split + min(j.split, more), u1 = u0 + per + (j.split < more);
    first = u0 + j.sub;
    n = j.NQ > 0 && u1 > first ? (u1 - first + j.warps - 1) / j.warps : 0;
  }
};

// Query row m of a lane: rows are beams x heads x tokens; its flat row of q's and out's [B, H, T].
__device__ __forceinline__ size_t share_row(const ShareGeo& a, const ShareJob& j, int m) {
  const int per = a.rf * a.T, w = m / per;
  return ((size_t)(j.b + w) * a.H + j.g * a.rf) * a.T + (m - w * per);
}
template <typename T>
__device__ __forceinline__ const T* share_query(const ShareGeo& a, const ShareJob& j, int m) {
  const int per = a.rf * a.T, w = m / per, h = (m - w * per) / a.T, t = m % a.T;
  return static_cast<const T*>(a.q) + (j.b + w) * a.qs[0] + (j.g * a.rf + h) * a.qs[1] + t * a.qs[2];
}

// Partial of one row: [m, l, -, -, O[D]], O relative to 2^m.
__device__ __forceinline__ float* share_part(float* part, const ShareGeo& a, int slot, size_t row) {
  return part + ((size_t)slot * a.B * a.H * a.T + row) * (a.D + 4);
}

constexpr int kShareWarps = 4;   // of a CTA that works with mma.sync
__device__ __forceinline__ void share_sync() { asm volatile("bar.sync 1, 128;\n" ::: "memory"); }

struct ShareJoin {
  float m[kShareWarps][16], l[kShareWarps][16];
};

// The results of a split's warps for its 16 rows, joined in warp order, as the split's partial.  `ring`: each warp's
// own shared memory, ring_bytes apart.
template <int D, int DT>
__device__ __forceinline__ void share_join_warps(const ShareGeo& a, const ShareJob& j, unsigned char* ring,
                                                 size_t ring_bytes, ShareJoin& join, float (&o)[DT][4], float m0, float m1,
                                                 float l0, float l1, float* part) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, t4 = lane & 3;
  if (j.warps == 1) {   // nothing to join
#pragma unroll
    for (int hr = 0; hr < 2; ++hr) {
      const int r = g8 + 8 * hr;
      if (r >= j.NQ) continue;
      float* p = share_part(part, a, j.slot, share_row(a, j, j.row0 + r));
      if (t4 == 0) *reinterpret_cast<float2*>(p) = hr ? make_float2(m1, l1) : make_float2(m0, l0);
#pragma unroll
      for (int jd = 0; jd < DT; ++jd)
        *reinterpret_cast<float2*>(p + 4 + jd * 8 + 2 * t4) = make_float2(o[jd][2 * hr], o[jd][2 * hr + 1]);
    }
    return;
  }
  float* wacc = reinterpret_cast<float*>(ring + warp * ring_bytes);
  if (t4 == 0) {
    join.m[warp][g8] = m0;
    join.l[warp][g8] = l0;
    join.m[warp][g8 + 8] = m1;
    join.l[warp][g8 + 8] = l1;
  }
#pragma unroll
  for (int jd = 0; jd < DT; ++jd) {
    const int c0 = jd * 8 + 2 * t4;
    *reinterpret_cast<float2*>(wacc + g8 * D + c0) = make_float2(o[jd][0], o[jd][1]);
    *reinterpret_cast<float2*>(wacc + (g8 + 8) * D + c0) = make_float2(o[jd][2], o[jd][3]);
  }
  share_sync();
  const int w0 = warp - j.sub;   // the split's first warp
  const int in = j.sub * 32 + lane;
  if (in < j.NQ) {
    float mw[kShareWarps], mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < kShareWarps; ++w) {
      mw[w] = w < j.warps ? join.m[(w0 + w) & 3][in] : -INFINITY;
      mx = fmaxf(mx, mw[w]);
    }
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < kShareWarps; ++w) {
      if (w >= j.warps) break;
      const float f = mw[w] == -INFINITY ? 0.f : exp2f(mw[w] - mx);
      l += join.l[w0 + w][in] * f;
      join.m[w0 + w][in] = f;
    }
    *reinterpret_cast<float2*>(share_part(part, a, j.slot, share_row(a, j, j.row0 + in))) = make_float2(mx, l);
  }
  share_sync();
  for (int x = in; x < j.NQ * (D / 4); x += j.warps * 32) {
    const int r = x / (D / 4), c = x % (D / 4) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kShareWarps; ++w) {
      if (w >= j.warps) break;
      const float4 y = *reinterpret_cast<const float4*>(ring + (w0 + w) * ring_bytes + (r * D + c) * 4);
      const float f = join.m[w0 + w][r];
      v.x = fmaf(y.x, f, v.x);
      v.y = fmaf(y.y, f, v.y);
      v.z = fmaf(y.z, f, v.z);
      v.w = fmaf(y.w, f, v.w);
    }
    *reinterpret_cast<float4*>(share_part(part, a, j.slot, share_row(a, j, j.row0 + r)) + 4 + c) = v;
  }
}

// Rows of a key tile that a query row of token `tok` sees: all of them, but of the new tokens under the causal mask
// those up to its own.
__device__ __forceinline__ unsigned share_see(const ShareGeo& a, bool fresh, int first, int rows, int tok) {
  const unsigned all = (1u << rows) - 1;
  if (!fresh || !a.causal) return all;
  const int n = tok - first + 1;
  return n <= 0 ? 0u : n >= rows ? all : (1u << n) - 1;
}

// ---------------------------------------------------------------- bf16: mma.sync, 16 query rows per CTA
// The 16 rows are the M of mma.sync.m16n8k16.  Each of the 4 warps streams 16-key tiles of its own through a
// private ring of cp.async stages (XOR-swizzled for ldmatrix); tiles do not cross segments.
constexpr int kShareStages = 3;

template <int D>
struct ShareShape {
  static constexpr int TS = 16, CPR = D / 8, KS = D / 16, DT = D / 8;
  static constexpr int STAGE_BYTES = 2 * TS * D * 2 + TS * 4;   // K, V, mass
  static constexpr size_t smem = (size_t)kShareWarps * kShareStages * STAGE_BYTES;
  __device__ __forceinline__ static int swz(int r, int c) {
    if (CPR >= 8) return c ^ (r & 7);
    return c ^ ((r * CPR / 8) & (CPR - 1));
  }
};

template <int D>
__device__ __forceinline__ void share_mma(const ShareGeo& a, const ShareJob& j, const logkv_prefix_t& pre,
                                          const __nv_bfloat16* rk, const __nv_bfloat16* rv, float* part,
                                          unsigned char* smem, ShareJoin& join) {
  using S = ShareShape<D>;
  using B16 = __nv_bfloat16;
  constexpr int TS = S::TS, CPR = S::CPR, KS = S::KS, DT = S::DT, ST = kShareStages;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, t4 = lane & 3;
  const ShareTiles u(j, TS);
  const int un = u.un, mine = u.n;
  unsigned char* wbase = smem + (size_t)warp * ST * S::STAGE_BYTES;
  const unsigned wbase_s = (unsigned)__cvta_generic_to_shared(wbase);
  // Segment 0 is the packed prefix with its mass terms, or the window's own rows; segment 1 the window's shared
  // rows, or the new tokens.
  const B16 *k0, *v0, *k1, *v1;
  long long ks1 = D, vs1 = D;
  const size_t win = ((size_t)j.b * a.G + j.g) * a.rcap * D;
  if (j.own) {
    k0 = rk + j.r0 * D, v0 = rv + j.r0 * D;
    k1 = static_cast<const B16*>(a.kn) + j.b * a.ks[0] + j.g * a.ks[1], ks1 = a.ks[2];
    v1 = static_cast<const B16*>(a.vn) + j.b * a.vs[0] + j.g * a.vs[1], vs1 = a.vs[2];
  } else {
    k0 = static_cast<const B16*>(pre.k) + j.r0 * D, v0 = static_cast<const B16*>(pre.v) + j.r0 * D;
    k1 = rk + win, v1 = rv + win;
  }
  const float* mass = j.own ? nullptr : pre.mass + j.r0;

  auto tile = [&](int t, int& first, int& rows) {
    const bool second = t >= un;
    first = (second ? t - un : t) * TS;
    rows = min(TS, (second ? j.n1 : j.n0) - first);
    return second;
  };
  auto issue = [&](int k, int stage) {
    if (k < mine) {
      int first, rows;
      const bool second = tile(u.first + k * j.warps, first, rows);
      const long long kst = second ? ks1 : D, vst = second ? vs1 : D;
      const B16* kb = (second ? k1 : k0) + first * kst;
      const B16* vb = (second ? v1 : v0) + first * vst;
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
        if (!second && mass && lane < rows) cp_async4(sm + lane, mass + first + lane);
        else sm[lane] = 0.f;
      }
    }
    cp_async_commit();
  };

#pragma unroll
  for (int k = 0; k < ST - 1; ++k) issue(k, k);
  int tok[2];   // tokens of the lane's rows g8 and g8 + 8
  unsigned qa[KS][4];
#pragma unroll
  for (int hr = 0; hr < 2; ++hr) {
    const int r = g8 + 8 * hr, m = j.row0 + max(0, min(r, j.NQ - 1));
    tok[hr] = m % a.T;
    const B16* qp = share_query<B16>(a, j, m);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qa[ks][hr] = r < j.NQ ? *reinterpret_cast<const unsigned*>(qp + ks * 16 + 2 * t4) : 0u;
      qa[ks][2 + hr] = r < j.NQ ? *reinterpret_cast<const unsigned*>(qp + ks * 16 + 2 * t4 + 8) : 0u;
    }
  }
  float o[DT][4];
#pragma unroll
  for (int i = 0; i < DT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  for (int k = 0; k < mine; ++k) {
    issue(k + ST - 1, (k + ST - 1) % ST);
    cp_async_wait<ST - 1>();
    __syncwarp();
    const int stage = k % ST;
    int first, rows;
    const bool fresh = tile(u.first + k * j.warps, first, rows) && j.own;
    unsigned char* st = wbase + (size_t)stage * S::STAGE_BYTES;
    const unsigned sk = wbase_s + stage * S::STAGE_BYTES, sv = sk + TS * D * 2;
    const float* sm = reinterpret_cast<const float*>(st + 2 * TS * D * 2);
    const unsigned see0 = share_see(a, fresh, first, rows, tok[0]), see1 = share_see(a, fresh, first, rows, tok[1]);
    unsigned poison = 0;   // new tokens whose V is not finite, taken out of the product below
    if (fresh && a.causal && a.T > 1) {
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
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = 8 * n + 2 * t4 + e;
        const float ms = sm[col] * a.mass_log2;
        sc[n][e] = see0 >> col & 1 ? fmaf(sc[n][e], a.scale_log2, ms) : -INFINITY;
        sc[n][2 + e] = see1 >> col & 1 ? fmaf(sc[n][2 + e], a.scale_log2, ms) : -INFINITY;
        mt0 = fmaxf(mt0, sc[n][e]);
        mt1 = fmaxf(mt1, sc[n][2 + e]);
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
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        p[n][e] = sc[n][e] == -INFINITY ? 0.f : exp2f(sc[n][e] - mn0);
        p[n][2 + e] = sc[n][2 + e] == -INFINITY ? 0.f : exp2f(sc[n][2 + e] - mn1);
        s0 += p[n][e];
        s1 += p[n][2 + e];
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
    // P as bf16 (the matrix instruction's operand type: off by at most 2^-8 relative, as much as the
    // output's own rounding); its row sums l stay float32 sums of the unrounded values.
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
  share_join_warps<D, DT>(a, j, smem, (size_t)ST * S::STAGE_BYTES, join, o, m0, m1, l0, l1, part);
}

template <int D, bool GROUPED>
__global__ void __launch_bounds__(kShareWarps * 32, D <= 128 ? 2 : 1)
    share_mma_kernel(ShareGeo a, logkv_prefix_t pre, const __nv_bfloat16* rk, const __nv_bfloat16* rv, float* part) {
  extern __shared__ uint4 smem4[];
  __shared__ ShareJoin join;
  ShareJob j = share_job<GROUPED>(a, pre);
  pdl_entry();
  share_keys(a, pre, ShareShape<D>::TS, j);
  if (j.split < j.ns) share_mma<D>(a, j, pre, rk, rv, part, reinterpret_cast<unsigned char*>(smem4), join);
}

// ---------------------------------------------------------------- bf16: tcgen05, up to 128 query rows per CTA
// Shared lanes of more than 16 rows, head dims 64 and 128.  The query rows (padded to the 128 rows of
// tcgen05.mma.cta_group::1.kind::f16) stay in shared memory; the CTA streams its split of the shared keys in units
// of 64:
//   warps 0-3  softmax, thread = query row = TMEM lane (warps past the last row leave at once);
//   warp 4     one thread issues S(r) = Q K(r)^T, then O += P(r-1) V(r-1);
//   warp 5     loads K and V: full tiles by TMA (128-byte swizzle, no multicast), a segment's last tile by cp.async
//              with zero fill.
// Tensor memory, 256 columns: two 64-column score buffers (P as bf16 over the first half of its own scores) and O.
// K and V have rings of their own: K(r) is free once its scores are done, V(r) once its product is.  Own lanes'
// CTAs of the launch work with mma.sync on warps 0-3.  Every wait is bounded; on expiry a role stops and the
// status gets bit 17.
constexpr int32_t kStatusShareTimeout = 1 << 17;
constexpr long long kShareWaitBudget = 4000000000LL;   // clock cycles (about 2 s)
constexpr int kShareTcThreads = 192;

template <int D>
struct ShareTcShape {
  static constexpr int TS = kTcTS, ST = D == 128 ? 2 : 4;
  static constexpr int MR = 2 * ST;   // mass stages, at least ST + 2
  static constexpr int Q_BYTES = (D / 64) * 128 * 128, KV_BYTES = (D / 64) * TS * 128;
  static constexpr int OFF_K = Q_BYTES, OFF_V = OFF_K + ST * KV_BYTES, OFF_M = OFF_V + ST * KV_BYTES;
  static constexpr size_t own = OFF_M + MR * TS * 4 + 1024;   // + alignment slack
  static constexpr size_t smem = own > ShareShape<D>::smem ? own : ShareShape<D>::smem;
  static constexpr uint32_t COLS = 256;
};

// K/V rows of the prefix and the window as tensor maps (64 x 64 boxes).
struct ShareMaps {
  CUtensorMap k[2];
  CUtensorMap v[2];
};

template <int D>
__global__ void __launch_bounds__(kShareTcThreads, 2)
    share_tc_kernel(ShareGeo a, logkv_prefix_t pre, const __nv_bfloat16* rk, const __nv_bfloat16* rv, float* part,
                    int32_t* status, const __grid_constant__ ShareMaps maps, int tma_mask) {
  using S = ShareTcShape<D>;
  using B16 = __nv_bfloat16;
  constexpr int TS = S::TS, ST = S::ST, MR = S::MR, CPR = D / 8;
  extern __shared__ uint4 smem4[];
  __shared__ ShareJoin join;
  __shared__ uint64_t q_full, k_full[ST], v_full[ST], k_empty[ST], v_empty[ST], m_full[MR], s_full[2], p_full[2],
      pv_done[2];
  __shared__ uint32_t sh_tmem;
  if (threadIdx.x < 4) tc::prefetch_tensormap(threadIdx.x < 2 ? &maps.k[threadIdx.x] : &maps.v[threadIdx.x - 2]);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  ShareJob j = share_job<true>(a, pre);
  const int live = (j.NQ + 31) / 32;   // softmax warps with rows
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
  pdl_entry();
  share_keys(a, pre, TS, j);
  unsigned char* raw = reinterpret_cast<unsigned char*>(smem4);
  if (j.own) {
    if (warp < kShareWarps) share_mma<D>(a, j, pre, rk, rv, part, raw, join);
    return;
  }
  if (j.split >= j.ns) return;
  const int up = (j.n0 + TS - 1) / TS, U = up + (j.n1 + TS - 1) / TS;
  const int per = U / j.ns, more = U - per * j.ns;   // the first `more` splits take a unit more
  const int u0 = per * j.split + min(j.split, more), n = per + (j.split < more);
  if (n == 0) {   // nothing shared at all: one split without keys
    for (int x = tid; x < j.NQ; x += kShareTcThreads) {
      float* pp = share_part(part, a, j.slot, share_row(a, j, j.row0 + x));
      *reinterpret_cast<float2*>(pp) = make_float2(-INFINITY, 0.f);
      for (int c = 0; c < D; c += 4) *reinterpret_cast<float4*>(pp + 4 + c) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    return;
  }
  unsigned char* base = raw + ((1024u - (tc::smem_u32(raw) & 1023u)) & 1023u);
  const uint32_t base_s = tc::smem_u32(base);
  if (warp == 0) {
    tc::tmem_alloc(&sh_tmem, S::COLS);
    tc::tmem_relinquish();
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = sh_tmem, t_o = tmem + 128u;
  auto t_s = [&](int r) { return tmem + 64u * (r & 1); };
  const size_t win = ((size_t)j.b * a.G + j.g) * a.rcap;
  auto unit = [&](int u, int& first, int& rows) {
    const int second = u >= up;
    first = (second ? u - up : u) * TS;
    rows = min(TS, (second ? j.n1 : j.n0) - first);
    return second;
  };
  auto fail = [&]() {
    if (status) atomicOr(status, kStatusShareTimeout);
  };

  if (warp == 5) {
    // ------------------------------------------------ loader
    auto row_of = [&](int seg, int first) { return (seg ? win : j.r0) + first; };
    // Key i's mass of unit r: read a unit ahead and not touched (so not waited for) until it is stored.
    auto mass_of = [&](int r, int i) {
      int first, rows;
      const int seg = unit(u0 + r, first, rows);
      return !seg && i < rows ? pre.mass[row_of(0, first) + i] : 0.f;
    };
    auto load = [&](int r, bool is_v) {
      const int st = r % ST;
      uint64_t* empty = is_v ? &v_empty[st] : &k_empty[st];
      uint64_t* full = is_v ? &v_full[st] : &k_full[st];
      if (r >= ST && !__all_sync(0xffffffffu, tc::mbar_wait(empty, (r / ST - 1) & 1, kShareWaitBudget))) return false;
      int first, rows;
      const int seg = unit(u0 + r, first, rows);
      unsigned char* dst = base + (is_v ? S::OFF_V : S::OFF_K) + st * S::KV_BYTES;
      if (rows == TS && (tma_mask >> seg & 1)) {
        if (lane == 0) {
          tc::fence_proxy_async();   // earlier plain stores to this stage before the asynchronous ones
          tc::mbar_arrive_expect_tx(full, S::KV_BYTES);
          const CUtensorMap* map = is_v ? &maps.v[seg] : &maps.k[seg];
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
            tc::tma_load_2d(tc::smem_u32(dst) + c * (TS * 128), map, c * 64, (int)row_of(seg, first), full);
        }
        return true;
      }
      const B16* src = (seg ? (is_v ? rv : rk) : static_cast<const B16*>(is_v ? pre.v : pre.k)) + row_of(seg, first) * D;
      for (int flat = lane; flat < TS * CPR; flat += 32) {
        const int i = flat / CPR, c = flat % CPR;
        unsigned char* d = dst + (c >> 3) * (TS * 128) + i * 128 + (((c & 7) ^ (i & 7)) << 4);
        if (i < rows) cp_async16(d, src + i * D + c * 8);
        else *reinterpret_cast<uint4*>(d) = make_uint4(0, 0, 0, 0);
      }
      cp_async_commit();
      cp_async_wait<0>();
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
      bool ok = tc::mbar_wait(&q_full, 0, kShareWaitBudget);
      for (int r = 0; ok && r <= n; ++r) {
        if (r < n) {
          const int st = r % ST;
          // Scores r overwrite P(r - 2): its product is done.
          ok = tc::mbar_wait(&k_full[st], (r / ST) & 1, kShareWaitBudget) &&
               (r < 2 || tc::mbar_wait(&pv_done[r & 1], (r / 2 - 1) & 1, kShareWaitBudget));
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
          ok = tc::mbar_wait(&v_full[st], (v / ST) & 1, kShareWaitBudget) &&
               tc::mbar_wait(&p_full[v & 1], (v / 2) & 1, kShareWaitBudget);
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
    const bool in = tid < j.NQ;
    const int m = j.row0 + min(tid, j.NQ - 1);
    {
      const B16* qp = share_query<B16>(a, j, m);
#pragma unroll
      for (int c = 0; c < CPR; ++c) {
        unsigned char* d = base + (c >> 3) * (128 * 128) + tid * 128 + (((c & 7) ^ (tid & 7)) << 4);
        if (in) cp_async16(d, qp + c * 8);
        else *reinterpret_cast<uint4*>(d) = make_uint4(0, 0, 0, 0);
      }
      cp_async_commit();
      cp_async_wait<0>();
      tc::fence_proxy_async();
      tc::mbar_arrive(&q_full);
    }
    float m_used = -INFINITY, l = 0.f;
    bool ok = true;
    for (int r = 0; r < n; ++r) {
      int first, rows;
      unit(u0 + r, first, rows);
      ok = __all_sync(0xffffffffu, tc::mbar_wait(&m_full[r % MR], (r / MR) & 1, kShareWaitBudget) &&
                                       tc::mbar_wait(&s_full[r & 1], (r / 2) & 1, kShareWaitBudget));
      if (!ok) break;
      tc::fence_after();
      const float* sm = reinterpret_cast<const float*>(base + S::OFF_M) + (r % MR) * TS;
      float sv[TS];
      {
        uint32_t r64[64];
        tc::tmem_ld64(t_s(r) + lane_off, r64);
#pragma unroll
        for (int i = 0; i < TS; ++i) sv[i] = __uint_as_float(r64[i]);
      }
      float mt = -INFINITY;
      const uint64_t c2 = tc::f2pack(a.scale_log2, a.scale_log2);
#pragma unroll
      for (int i = 0; i < TS; i += 4) {
        const float4 m4 = *reinterpret_cast<const float4*>(sm + i);
        tc::f2unpack(tc::ffma2(tc::f2pack(sv[i], sv[i + 1]), c2, tc::f2pack(m4.x, m4.y)), sv[i], sv[i + 1]);
        tc::f2unpack(tc::ffma2(tc::f2pack(sv[i + 2], sv[i + 3]), c2, tc::f2pack(m4.z, m4.w)), sv[i + 2], sv[i + 3]);
      }
      if (rows < TS) {
#pragma unroll
        for (int i = 0; i < TS; ++i) sv[i] = i < rows ? sv[i] : -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < TS; i += 4) mt = fmaxf(mt, fmaxf(fmaxf(sv[i], sv[i + 1]), fmaxf(sv[i + 2], sv[i + 3])));
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
      for (int i = 0; i < 32; ++i) {
        float x0, x1;
        tc::f2unpack(tc::fadd2(tc::f2pack(sv[2 * i], sv[2 * i + 1]), nm2), x0, x1);
        const float p0 = tc::ex2(x0), p1 = tc::ex2(x1);
        ps2 = tc::fadd2(ps2, tc::f2pack(p0, p1));
        pk[i] = pack_bf16x2(p0, p1);   // the matrix instruction's operand type; l sums the unrounded values
      }
      float ps0, ps1;
      tc::f2unpack(ps2, ps0, ps1);
      l = l * alpha + (ps0 + ps1);
      if (r > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
        ok = __all_sync(0xffffffffu, tc::mbar_wait(&pv_done[(r - 1) & 1], ((r - 1) / 2) & 1, kShareWaitBudget));
        if (!ok) break;
        tc::fence_after();
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += 32) {
          uint32_t r32[32];
          tc::tmem_ld32(t_o + lane_off + c0, r32);
#pragma unroll
          for (int i = 0; i < 32; ++i) r32[i] = __float_as_uint(__uint_as_float(r32[i]) * alpha);
          tc::tmem_st32(t_o + lane_off + c0, r32);
        }
      }
      tc::tmem_st32(t_s(r) + lane_off, pk);
      tc::fence_before();
      tc::mbar_arrive(&p_full[r & 1]);
    }
    if (ok) ok = __all_sync(0xffffffffu, tc::mbar_wait(&pv_done[(n - 1) & 1], ((n - 1) / 2) & 1, kShareWaitBudget));
    if (!ok) {
      if (lane == 0) fail();
    } else {
      tc::fence_after();
      float* pp = share_part(part, a, j.slot, share_row(a, j, m));
      if (in) *reinterpret_cast<float2*>(pp) = make_float2(m_used, l);
#pragma unroll 1
      for (int c0 = 0; c0 < D; c0 += 32) {
        uint32_t r32[32];
        tc::tmem_ld32(t_o + lane_off + c0, r32);
        if (!in) continue;
#pragma unroll
        for (int i = 0; i < 32; i += 4)
          *reinterpret_cast<float4*>(pp + 4 + c0 + i) =
              make_float4(__uint_as_float(r32[i]), __uint_as_float(r32[i + 1]), __uint_as_float(r32[i + 2]),
                          __uint_as_float(r32[i + 3]));
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
// As the bf16 kernel with mma.sync.m16n8k8 (tf32), every float32 operand split in two.  K and V rows are padded by
// 16 bytes, so that the fragments' reads fall into 32 different banks.
template <int D>
struct ShareF32Shape {
  static constexpr int TS = 16, LD = D + 4, KS = D / 8, DT = D / 8, CPR = D / 4;
  static constexpr int ST = D == 64 ? 2 : 3;   // two CTAs per SM up to 64 features, one at 128
  static constexpr int STAGE_BYTES = 2 * TS * LD * 4 + TS * 4;   // K, V, mass
  static constexpr size_t smem = (size_t)kShareWarps * ST * STAGE_BYTES;
  static constexpr int CTAS = D <= 64 ? 2 : 1;   // per SM
};

template <int D, bool GROUPED>
__global__ void __launch_bounds__(kShareWarps * 32, ShareF32Shape<D>::CTAS)
    share_f32_kernel(ShareGeo a, logkv_prefix_t pre, const float* rk, const float* rv, float* part) {
  using S = ShareF32Shape<D>;
  constexpr int TS = S::TS, LD = S::LD, KS = S::KS, DT = S::DT, CPR = S::CPR, ST = S::ST;
  extern __shared__ uint4 smem4[];
  __shared__ ShareJoin join;
  ShareJob j = share_job<GROUPED>(a, pre);
  pdl_entry();
  share_keys(a, pre, TS, j);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, t4 = lane & 3;
  if (j.split >= j.ns) return;
  const ShareTiles u(j, TS);
  const int un = u.un, mine = u.n;
  unsigned char* wbase = reinterpret_cast<unsigned char*>(smem4) + (size_t)warp * ST * S::STAGE_BYTES;
  const float *k0, *v0, *k1, *v1;
  long long ks1 = D, vs1 = D;
  const size_t win = ((size_t)j.b * a.G + j.g) * a.rcap * D;
  if (j.own) {
    k0 = rk + j.r0 * D, v0 = rv + j.r0 * D;
    k1 = static_cast<const float*>(a.kn) + j.b * a.ks[0] + j.g * a.ks[1], ks1 = a.ks[2];
    v1 = static_cast<const float*>(a.vn) + j.b * a.vs[0] + j.g * a.vs[1], vs1 = a.vs[2];
  } else {
    k0 = static_cast<const float*>(pre.k) + j.r0 * D, v0 = static_cast<const float*>(pre.v) + j.r0 * D;
    k1 = rk + win, v1 = rv + win;
  }
  const float* mass = j.own ? nullptr : pre.mass + j.r0;
  auto tile = [&](int t, int& first, int& rows) {
    const bool second = t >= un;
    first = (second ? t - un : t) * TS;
    rows = min(TS, (second ? j.n1 : j.n0) - first);
    return second;
  };
  auto issue = [&](int k, int stage) {
    if (k < mine) {
      int first, rows;
      const bool second = tile(u.first + k * j.warps, first, rows);
      const long long kst = second ? ks1 : D, vst = second ? vs1 : D;
      const float* kb = (second ? k1 : k0) + first * kst;
      const float* vb = (second ? v1 : v0) + first * vst;
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
        if (!second && mass && lane < rows) cp_async4(sm + lane, mass + first + lane);
        else sm[lane] = 0.f;
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int k = 0; k < ST - 1; ++k) issue(k, k);
  int tok[2];   // tokens of the lane's rows g8 and g8 + 8
  float qf[KS][4];   // A fragments: (g8, t4), (g8 + 8, t4), (g8, t4 + 4), (g8 + 8, t4 + 4)
#pragma unroll
  for (int hr = 0; hr < 2; ++hr) {
    const int r = g8 + 8 * hr, m = j.row0 + max(0, min(r, j.NQ - 1));
    tok[hr] = m % a.T;
    const float* qp = share_query<float>(a, j, m);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[ks][hr] = r < j.NQ ? qp[ks * 8 + t4] : 0.f;
      qf[ks][2 + hr] = r < j.NQ ? qp[ks * 8 + t4 + 4] : 0.f;
    }
  }
  float o[DT][4];
#pragma unroll
  for (int i = 0; i < DT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  for (int k = 0; k < mine; ++k) {
    issue(k + ST - 1, (k + ST - 1) % ST);
    cp_async_wait<ST - 1>();
    __syncwarp();
    int first, rows;
    const bool fresh = tile(u.first + k * j.warps, first, rows) && j.own;
    float* sk = reinterpret_cast<float*>(wbase + (size_t)(k % ST) * S::STAGE_BYTES);
    float* sv = sk + TS * LD;
    const float* sm = sv + TS * LD;
    const unsigned see0 = share_see(a, fresh, first, rows, tok[0]), see1 = share_see(a, fresh, first, rows, tok[1]);
    unsigned poison = 0;   // new tokens whose V is not finite, taken out of the product below
    if (fresh && a.causal && a.T > 1) {
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
      for (int n = 0; n < 2; ++n)
        mma_split(sc[n], ah, al, sk[(8 * n + g8) * LD + 8 * ks + t4], sk[(8 * n + g8) * LD + 8 * ks + t4 + 4]);
    }
    float mt0 = -INFINITY, mt1 = -INFINITY;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = 8 * n + 2 * t4 + e;
        const float ms = sm[col] * a.mass_log2;
        sc[n][e] = see0 >> col & 1 ? fmaf(sc[n][e], a.scale_log2, ms) : -INFINITY;
        sc[n][2 + e] = see1 >> col & 1 ? fmaf(sc[n][2 + e], a.scale_log2, ms) : -INFINITY;
        mt0 = fmaxf(mt0, sc[n][e]);
        mt1 = fmaxf(mt1, sc[n][2 + e]);
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
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        p[n][e] = sc[n][e] == -INFINITY ? 0.f : exp2f(sc[n][e] - mn0);
        p[n][2 + e] = sc[n][2 + e] == -INFINITY ? 0.f : exp2f(sc[n][2 + e] - mn1);
        s0 += p[n][e];
        s1 += p[n][2 + e];
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
    // O += P V, eight keys at a time: key 8 n + 2 t4 + e is index t4 + 4 e of the product, which makes the
    // scores' fragment P's.
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      unsigned ph[4], pl[4];
      split_tf32(p[n][0], ph[0], pl[0]);
      split_tf32(p[n][2], ph[1], pl[1]);
      split_tf32(p[n][1], ph[2], pl[2]);
      split_tf32(p[n][3], ph[3], pl[3]);
      const float* vr = sv + (8 * n + 2 * t4) * LD + g8;
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
  share_join_warps<D, DT>(a, j, reinterpret_cast<unsigned char*>(smem4), (size_t)ST * S::STAGE_BYTES, join, o, m0, m1,
                          l0, l1, part);
}

// ---------------------------------------------------------------- combine
// WPR warps per output row (1 or 4): each joins its share of the row's partials (the shared splits, then the own
// ones), NB at a time with all of their loads in flight, then the warps in order.  TS: the key tile of the kernel that
// wrote the shared partials.  Index arithmetic alone stands before the wait: the prefix's length comes from a kernel in
// front of the attention's, and what those wrote is visible here only behind it.
template <typename T, int D, int TS, int WPR>
__global__ void __launch_bounds__(128) share_combine_kernel(ShareGeo a, logkv_prefix_t pre, const float* part, T* out) {
  constexpr int PER = (D + 127) / 128, NB = D > 128 ? 4 : 10;
  __shared__ float sh[4][2 + D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp % WPR;
  const size_t row = (size_t)blockIdx.x * (4 / WPR) + warp / WPR;
  const bool live = WPR > 1 || row < (size_t)a.B * a.H * a.T;
  const int bh = (int)(row / a.T), ln = bh / a.H / a.W * a.W * a.G + bh % a.H / a.rf, window = (a.w0 + TS - 1) / TS;
  const size_t stride = (size_t)a.B * a.H * a.T * (D + 4);
  const float* p0 = part + row * (D + 4);
  pdl_entry();
  if (!live) return;
  const int shared = share_splits(a, (share_prefix_length(pre, ln) + TS - 1) / TS + window, TS);
  const int ns = shared + a.nown, skip = a.nsplit - shared;   // partials; unused slots between the two kinds
  auto at = [&](int s) { return p0 + (size_t)(s < shared ? s : s + skip) * stride; };
  float m = -INFINITY, l = 0.f;
  float4 o[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  const int share = (ns + WPR - 1) / WPR, end = min(ns, (sub + 1) * share);
  for (int s0 = sub * share; s0 < end; s0 += NB) {
    float2 ml[NB];
    float4 v[NB][PER];
#pragma unroll
    for (int s = 0; s < NB; ++s) {
      const bool in = s0 + s < end;
      const float* p = at(in ? s0 + s : s0);
      ml[s] = in ? *reinterpret_cast<const float2*>(p) : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int c = 4 * (lane + 32 * k);
        v[s][k] = in && c < D ? *reinterpret_cast<const float4*>(p + 4 + c) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
    float mn = m;
#pragma unroll
    for (int s = 0; s < NB; ++s) mn = fmaxf(mn, ml[s].x);
    const float al = m == -INFINITY ? 0.f : exp2f(m - mn);
    l *= al;
    m = mn;
#pragma unroll
    for (int k = 0; k < PER; ++k) o[k] = make_float4(o[k].x * al, o[k].y * al, o[k].z * al, o[k].w * al);
#pragma unroll
    for (int s = 0; s < NB; ++s) {
      const float w = ml[s].x == -INFINITY ? 0.f : exp2f(ml[s].x - mn);
      l = fmaf(ml[s].y, w, l);
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        o[k].x = fmaf(v[s][k].x, w, o[k].x);
        o[k].y = fmaf(v[s][k].y, w, o[k].y);
        o[k].z = fmaf(v[s][k].z, w, o[k].z);
        o[k].w = fmaf(v[s][k].w, w, o[k].w);
      }
    }
  }
  if (WPR > 1) {
    if (lane == 0) {
      sh[warp][0] = m;
      sh[warp][1] = l;
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
    for (int w = 0; w < WPR; ++w) m = fmaxf(m, sh[w][0]);
    for (int d = threadIdx.x; d < D; d += 128) {
      float L = 0.f, x = 0.f;
#pragma unroll
      for (int w = 0; w < WPR; ++w) {
        const float f = sh[w][0] == -INFINITY ? 0.f : exp2f(sh[w][0] - m);
        L += sh[w][1] * f;
        x += sh[w][2 + d] * f;
      }
      Elem<T>::store(out + row * D + d, x / L);
    }
    return;
  }
  const float inv = 1.f / l;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int c = 4 * (lane + 32 * k);
    if (c < D) {
      T* dst = out + row * D + c;
      Elem<T>::store(dst, o[k].x * inv);
      Elem<T>::store(dst + 1, o[k].y * inv);
      Elem<T>::store(dst + 2, o[k].z * inv);
      Elem<T>::store(dst + 3, o[k].w * inv);
    }
  }
}

// ---------------------------------------------------------------- host side
struct SharePlan {
  int tile_rows, tiles, own_tiles, nsplit, upw, nown, own_warps, slots;
  long long own_work;
  bool tc;
};

static SharePlan share_plan(const logkv_layout_t& l, const logkv_shared_args_t& x, int prefix_capacity) {
  SharePlan p;
  const bool f32 = l.dtype == LOGKV_DTYPE_F32;
  const long long own_rows = (long long)(x.heads / l.groups) * x.q_tokens, rows = own_rows * x.beams;
  p.tc = !f32 && (l.dim == 64 || l.dim == 128) && rows > 16;
  const int most = p.tc ? 128 : 16;
  p.tiles = (int)((rows + most - 1) / most);
  p.tile_rows = p.tc ? (int)((rows + p.tiles - 1) / p.tiles) : most;
  p.own_tiles = (int)((own_rows + 15) / 16);
  const int ts = p.tc ? kTcTS : 16;
  p.upw = p.tc ? 2 : kShareWarps;
  p.slots = 148 * ((f32 && l.dim > 64) || l.dim > 128 ? 1 : 2);
  const long long own = (long long)l.batch * l.groups * p.own_tiles;
  const long long shared_ctas = (long long)l.batch / x.beams * l.groups * p.tiles;
  // A second split of an own lane (a key tile per warp at least) only while they leave half of the SMs.
  const int own_keys = x.recent_count - x.window_from + x.tokens;
  p.nown = (int)std::max(1LL, std::min<long long>(own_keys / 16 / kShareWarps, p.slots / 2 / own));
  // The grid holds the splits of a full prefix; a shorter one leaves some unused.  Starting a warp on an own lane
  // weighs as much as some 50 keys of a CTA.
  const long long units = (prefix_capacity + x.window_from) / ts + 2, work = units * ts * shared_ctas;
  auto own_work = [&](int warps) { return own * p.nown * (own_keys / p.nown + 50LL * warps); };
  // Warps to an own lane: as many as fit into its kind's share of the SMs, a prefix taken to fill 0.6 of its capacity,
  // and so many that none has more than eight key tiles (one warp's 16 take 22 us: 512 lanes of 242 keys beside 64 shared
  // ones 59.6, 60.1, 61.3 us with 4, 2 and 1).
  // Own parts of 64 keys beside 3.3K shared ones in us with 4, 2 and 1: 256 lanes beside 64 shared ones 30, 31, 26.5;
  // 1024 beside 64 67, 54, 44; 32 beside 8 12.4, 14.2, 14.1.  405 keys, 480 lanes, hardly any shared ones: 33, 31, 39.
  p.own_warps = 4;
  while (p.nown == 1 && p.own_warps > 1 && own_keys <= 8 * 16 * p.own_warps / 2 &&
         own * p.own_warps / 4 > p.slots * own_work(p.own_warps) / (work * 6 / 10 + own_work(p.own_warps)))
    p.own_warps /= 2;
  p.own_work = own_work(p.own_warps);
  long long splits = std::min((2 * p.slots * work / (work + p.own_work) + shared_ctas) / (2 * shared_ctas),
                              std::max(1LL, p.slots / shared_ctas));
  // A few splits fewer let all CTAs run at once (32 own ones beside 8 lanes: 13.3 us with 33 splits, 13.6 with 34).
  const long long beside = (p.slots - (own * p.nown * p.own_warps + 3) / 4) / shared_ctas;
  if (beside < splits && beside >= splits - splits / 8) splits = beside;
  p.nsplit = (int)std::max(1LL, std::min(splits, units / p.upw));
  return p;
}

static int check_shared(const logkv_layout_t* l, const logkv_shared_args_t* x, int prefix_capacity) {
  const int rc = check_layout(l);
  if (rc) return rc;
  if (!x) return LOGKV_E_POINTER;
  const bool dim = l->dim == 16 || l->dim == 32 || l->dim == 64 || l->dim == 128 ||
                   (l->dim == 256 && l->dtype == LOGKV_DTYPE_BF16);
  if (!dim || x->heads < l->groups || x->heads % l->groups || x->beams < 1 || l->batch % x->beams || x->q_tokens < 1 ||
      x->tokens < x->q_tokens || (x->causal && x->tokens != x->q_tokens) || x->recent_count < 0 ||
      x->recent_count > l->recent_capacity || x->window_from < 0 || x->window_from > x->recent_count || prefix_capacity < 0)
    return LOGKV_E_SHAPE;
  // Query rows of a lane and CTAs of the grid.
  if ((long long)(x->heads / l->groups) * x->q_tokens * x->beams > (1 << 20)) return LOGKV_E_SHAPE;
  const SharePlan p = share_plan(*l, *x, prefix_capacity);
  const long long ctas = (long long)l->batch / x->beams * l->groups * p.tiles * p.nsplit +
                         (long long)l->batch * l->groups * p.own_tiles * p.nown;
  return ctas > 0x7fffffffLL || (long long)l->batch * x->heads * x->q_tokens > 0x7fffffffLL ? LOGKV_E_SHAPE : LOGKV_OK;
}

template <typename T, int D, int TS>
static void launch_share_combine(const ShareGeo& a, const logkv_prefix_t& pre, const float* part, void* out,
                                 cudaStream_t st) {
  const size_t rows = (size_t)a.B * a.H * a.T;
  T* o = static_cast<T*>(out);
  // Four warps to a row where there are many partials and few rows: 64 rows of 32 partials 3 us less; with 1920 rows
  // of 13 the extra warps only wait (27 us in all against 17).
  if (a.nsplit + a.nown > 8 && rows <= 148 * 8)
    launch_pdl(share_combine_kernel<T, D, TS, 4>, dim3((unsigned)rows), 128, 0, st, a, pre, part, o);
  else
    launch_pdl(share_combine_kernel<T, D, TS, 1>, dim3((unsigned)((rows + 3) / 4)), 128, 0, st, a, pre, part, o);
}

static dim3 share_grid(const ShareGeo& a) {
  return dim3((unsigned)(a.shared_lanes * a.nsplit * a.tiles +
                         ((long long)a.own_lanes * a.nown * a.own_tiles * a.own_warps + 3) / 4));
}

template <int D>
static int launch_share_bf16(const ShareGeo& a, const logkv_prefix_t& pre, const logkv_state_t& s, void* out, float* part,
                             cudaStream_t st) {
  using B16 = __nv_bfloat16;
  const auto kern = a.own_warps < 4 ? share_mma_kernel<D, true> : share_mma_kernel<D, false>;
  const int e = a.own_warps < 4 ? smem_limit_once<share_mma_kernel<D, true>>(ShareShape<D>::smem)
                                : smem_limit_once<share_mma_kernel<D, false>>(ShareShape<D>::smem);
  if (e) return e;
  launch_pdl(kern, share_grid(a), kShareWarps * 32, ShareShape<D>::smem, st, a, pre,
             static_cast<const B16*>(s.recent_k), static_cast<const B16*>(s.recent_v), part);
  launch_share_combine<B16, D, 16>(a, pre, part, out, st);
  return launch_status();
}

template <int D>
static int launch_share_tc(const ShareGeo& a, const logkv_prefix_t& pre, const logkv_state_t& s, void* out, float* part,
                           int32_t* status, cudaStream_t st) {
  using B16 = __nv_bfloat16;
  if (const int e = smem_limit_once<share_tc_kernel<D>>(ShareTcShape<D>::smem)) return e;
  ShareMaps maps;
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
  launch_pdl(share_tc_kernel<D>, share_grid(a), kShareTcThreads, ShareTcShape<D>::smem, st, a, pre,
             static_cast<const B16*>(s.recent_k), static_cast<const B16*>(s.recent_v), part, status, maps, mask);
  launch_share_combine<B16, D, kTcTS>(a, pre, part, out, st);
  return launch_status();
}

template <int D>
static int launch_share_f32(const ShareGeo& a, const logkv_prefix_t& pre, const logkv_state_t& s, void* out, float* part,
                            cudaStream_t st) {
  const auto kern = a.own_warps < 4 ? share_f32_kernel<D, true> : share_f32_kernel<D, false>;
  const int e = a.own_warps < 4 ? smem_limit_once<share_f32_kernel<D, true>>(ShareF32Shape<D>::smem)
                                : smem_limit_once<share_f32_kernel<D, false>>(ShareF32Shape<D>::smem);
  if (e) return e;
  launch_pdl(kern, share_grid(a), kShareWarps * 32, ShareF32Shape<D>::smem, st, a, pre,
             static_cast<const float*>(s.recent_k), static_cast<const float*>(s.recent_v), part);
  launch_share_combine<float, D, 16>(a, pre, part, out, st);
  return launch_status();
}

}  // namespace logkv

using namespace logkv;

extern "C" {

LOGKV_API size_t logkv_shared_attention_workspace_bytes(const logkv_layout_t* layout, const logkv_shared_args_t* args,
                                                        int32_t prefix_capacity) {
  if (check_shared(layout, args, prefix_capacity)) return 0;
  const SharePlan p = share_plan(*layout, *args, prefix_capacity);
  return (size_t)(p.nsplit + p.nown) * layout->batch * args->heads * args->q_tokens * (layout->dim + 4) * sizeof(float);
}

LOGKV_API int logkv_shared_attention(const logkv_layout_t* layout, const logkv_state_t* state,
                                     const logkv_prefix_t* prefix, const logkv_shared_args_t* x, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  if (!layout || !state || !prefix || !x) return LOGKV_E_POINTER;
  const int rc = check_shared(layout, x, prefix->capacity);
  if (rc) return rc;
  auto at = [](const void* p, uintptr_t n) { return p && (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  auto a16 = [&](const void* p) { return at(p, 16); };
  if (!a16(x->q) || !a16(x->k_new) || !a16(x->v_new) || !a16(x->out) || !a16(workspace) || !a16(state->recent_k) ||
      !a16(state->recent_v) || !a16(prefix->k) || !a16(prefix->v) || !at(prefix->mass, 4) || !at(prefix->length, 4))
    return LOGKV_E_POINTER;
  const long long e = (long long)esize_of(layout->dtype);
  ShareGeo a{};
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = x->q_strides[i];
    a.ks[i] = x->k_strides[i];
    a.vs[i] = x->v_strides[i];
    if (a.qs[i] * e % 16 || a.ks[i] * e % 16 || a.vs[i] * e % 16) return LOGKV_E_POINTER;
  }
  if (workspace_bytes < logkv_shared_attention_workspace_bytes(layout, x, prefix->capacity)) return LOGKV_E_WORKSPACE;
  const SharePlan p = share_plan(*layout, *x, prefix->capacity);
  a.B = layout->batch;
  a.G = layout->groups;
  a.H = x->heads;
  a.rf = a.H / a.G;
  a.T = x->q_tokens;
  a.Tk = x->tokens;
  a.W = x->beams;
  a.D = layout->dim;
  a.rcap = layout->recent_capacity;
  a.rcount = x->recent_count;
  a.w0 = x->window_from;
  a.causal = x->causal;
  a.nsplit = p.nsplit;
  a.upw = p.upw;
  a.nown = p.nown;
  a.own_warps = p.own_warps;
  a.shared_lanes = a.B / a.W * a.G;
  a.own_lanes = a.B * a.G;
  a.tiles = p.tiles;
  a.tile_rows = p.tile_rows;
  a.own_tiles = p.own_tiles;
  a.slots = p.slots;
  a.own_work = (float)p.own_work;
  a.scale_log2 = x->scale * 1.4426950408889634f;
  a.mass_log2 = x->qx * a.scale_log2;
  a.q = x->q;
  a.kn = x->k_new;
  a.vn = x->v_new;
  float* part = static_cast<float*>(workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p.tc) {
    if (layout->dim == 64) return launch_share_tc<64>(a, *prefix, *state, x->out, part, x->status, st);
    return launch_share_tc<128>(a, *prefix, *state, x->out, part, x->status, st);
  }
  if (layout->dtype == LOGKV_DTYPE_BF16) {
    switch (layout->dim) {
      case 16: return launch_share_bf16<16>(a, *prefix, *state, x->out, part, st);
      case 32: return launch_share_bf16<32>(a, *prefix, *state, x->out, part, st);
      case 64: return launch_share_bf16<64>(a, *prefix, *state, x->out, part, st);
      case 128: return launch_share_bf16<128>(a, *prefix, *state, x->out, part, st);
      default: return launch_share_bf16<256>(a, *prefix, *state, x->out, part, st);
    }
  }
  switch (layout->dim) {
    case 16: return launch_share_f32<16>(a, *prefix, *state, x->out, part, st);
    case 32: return launch_share_f32<32>(a, *prefix, *state, x->out, part, st);
    case 64: return launch_share_f32<64>(a, *prefix, *state, x->out, part, st);
    default: return launch_share_f32<128>(a, *prefix, *state, x->out, part, st);
  }
}

}  // extern "C"
