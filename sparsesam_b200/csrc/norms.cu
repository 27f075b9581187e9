// Group normalisation with an activation on channels-last maps, forward and
// backward, and the backward pass of the channel LayerNorm (+ GELU) of half rows.
//
//   xh = (x - mu) rstd,  z = xh w + b,  y = act(z),  rstd = 1 / sqrt(var + eps)
//   g = dy act'(z),  db = sum g,  dw = sum g xh,
//   dx = rstd (g w - mean(g w) - xh mean(g w xh))      (means over what mu is a mean of)
//
// mu and var are over the positions and channels of one group of one sample
// (GroupNorm) or over the channels of one row (LayerNorm). Means and squared
// deviations are merged pairwise from short exact batches (Chan, Golub, LeVeque,
// "Updating formulae and a pairwise algorithm for computing sample variances",
// 1979), so a mean far from zero or an outlier costs no digits of the variance.
// Everything is computed in fp32 and rounded once, to x's type, at the end.
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "host_util.h"

namespace ssam {

enum { kActNone = 0, kActRelu = 1, kActGelu = 2, kActSilu = 3 };

// act(z) and act'(z). EXACT (fp32 maps) takes the full-precision functions. The half
// types take erf from Abramowitz & Stegun 7.1.26 (as gelu_exact, |error| 1.5e-7; the
// exponential of erf is the one of GELU's slope) and the approximate exponential and
// division: a thousandth of the output's rounding, and 2 to 3 times fewer instructions,
// which is what bounded these kernels (GELU apply of 16 x 256 x 256 x 64: 108 us exact).
template <int ACT, bool EXACT>
__device__ __forceinline__ float act_value(float z) {
  if (ACT == kActRelu) return z < 0.f ? 0.f : z;  // NaN stays NaN
  if (ACT == kActGelu) return EXACT ? 0.5f * z * (1.f + erff(z * 0.70710678118654752440f)) : gelu_exact(z);
  if (ACT == kActSilu) return EXACT ? z / (1.f + expf(-z)) : __fdividef(z, 1.f + __expf(-z));
  return z;
}
// GELU'(z) = Phi(z) + z phi(z); with u = |z| / sqrt 2 and q the polynomial part of 7.1.26,
// Phi = 1/2 + sign(z) (1/2 - q exp(-u^2) / 2).
__device__ __forceinline__ float gelu_slope_fast(float z) {
  const float u = fabsf(z) * 0.70710678118654752440f;
  float t, e;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(0.3275911f, u, 1.0f)));
  const float half_q =
      fmaf(fmaf(fmaf(fmaf(0.5307027145f, t, -0.7265760135f), t, 0.7107068705f), t, -0.142248368f), t, 0.127414796f) * t;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(u * u * -1.4426950408889634f));
  const float tail = half_q * e;
  return fmaf(z * 0.39894228040143267794f, e, z >= 0.f ? 1.f - tail : tail);
}
template <int ACT, bool EXACT>
__device__ __forceinline__ float act_slope(float z) {
  if (ACT == kActRelu) return z > 0.f ? 1.f : 0.f;
  if (ACT == kActGelu)
    return EXACT ? 0.5f * (1.f + erff(z * 0.70710678118654752440f)) + z * expf(-0.5f * z * z) * 0.39894228040143267794f
                 : gelu_slope_fast(z);
  if (ACT == kActSilu) {
    const float s = EXACT ? 1.f / (1.f + expf(-z)) : __fdividef(1.f, 1.f + __expf(-z));
    return s * (1.f + z * (1.f - s));
  }
  return 1.f;
}

// V consecutive channels (16 bytes) of a row as floats.
template <class T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int V = 4;
  static constexpr bool exact = true;
  static __device__ __forceinline__ void load(const float* p, float (&f)[4]) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
  }
  static __device__ __forceinline__ void store(float* p, const float (&f)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  }
};
template <>
struct Vec<__half> {
  static constexpr int V = 8;
  static constexpr bool exact = false;
  static __device__ __forceinline__ void load(const __half* p, float (&f)[8]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = v.x, f[2 * i + 1] = v.y;
    }
  }
  static __device__ __forceinline__ void store(__half* p, const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int V = 8;
  static constexpr bool exact = false;
  static __device__ __forceinline__ void load(const __nv_bfloat16* p, float (&f)[8]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&f)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                                              pack_bf16x2(f[6], f[7]));
  }
};
__device__ __forceinline__ void norm_store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void norm_store1(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void norm_store1(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// ---------------------------------------------------------------------------
// GroupNorm
//
// Threads of a block form `lanes` position lanes of `cols` 16-byte vector columns: a
// thread keeps its channels and walks positions. Two shapes of work:
//
//  * Resident (one launch, x read once): a cluster holds the positions of one sample and
//    one slab of whole groups in shared memory, reduces through distributed shared memory
//    and writes the result. A slab is at least 64 bytes wide, so that sectors are whole.
//  * Streamed (samples too large for that): a moments / sums kernel, then an apply kernel,
//    launched for as many samples at a time as stay in L2 between the two (48 MB), so
//    that HBM still sees x once. 16 x 256 x 256 x 64 bf16 GELU with gradients: 567 us when
//    both kernels ran over the whole batch, with the exact functions.
// ---------------------------------------------------------------------------
constexpr int kGnThreads = 256;
constexpr int kGnWarps = kGnThreads / 32;
constexpr int kGnBatch = 4;                     // positions loaded ahead; their moments are exact, then merged
constexpr int64_t kGnResident = 96 << 10;       // shared-memory bytes a resident block may hold (two blocks per SM)
constexpr int64_t kGnL2 = 48 << 20;             // bytes of a streamed batch of samples

// red[g * parts + i], i < parts: partial sums of vals[lane][C] over the lanes and the cg channels of
// group g. Ends with the block synchronised; the return value is `parts`. vals may be reused after it.
__device__ __forceinline__ int group_sums(const float* vals, int lanes, int C, int cg, float* red) {
  const int G = C / cg, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  int parts = 1;
  while (parts * 2 * G <= kGnWarps) parts *= 2;
  __syncthreads();
  for (int g = warp / parts; g < G; g += kGnWarps / parts) {
    float s = 0.f;
    for (int e = warp % parts * 32 + lane; e < lanes * cg; e += parts * 32) s += vals[e / cg * C + g * cg + e % cg];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) red[g * parts + warp % parts] = s;
  }
  __syncthreads();
  return parts;
}
__device__ __forceinline__ float sum_parts(const float* red, int g, int parts) {
  float s = 0.f;
  for (int i = 0; i < parts; ++i) s += red[g * parts + i];
  return s;
}

// A thread's running per-channel moments of n positions.
template <int V>
struct Running {
  float n = 0.f, mean[V], m2[V];
  __device__ __forceinline__ Running() {
#pragma unroll
    for (int i = 0; i < V; ++i) mean[i] = 0.f, m2[i] = 0.f;
  }
  // K loaded positions of which the first k >= 1 count (the others are zeros)
  template <int K>
  __device__ __forceinline__ void add(const float (&f)[K][V], int k) {
    const float kf = static_cast<float>(k), inv = __frcp_rn(kf), nn = n + kf, w = __fdividef(kf, nn), cw = n * w;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float s = 0.f, q = 0.f;
#pragma unroll
      for (int j = 0; j < K; ++j) s += f[j][i];
      s *= inv;
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const float d = j < k ? f[j][i] - s : 0.f;
        q = fmaf(d, d, q);
      }
      const float d = s - mean[i];
      mean[i] = fmaf(d, w, mean[i]);
      m2[i] += fmaf(d * d, cw, q);
    }
    n = nn;
  }
};

// Group means and squared deviations of a block's positions [len] from the threads' running moments:
// s_mean[g], s_m2[g]. vals: [lanes][C], red: [max(G, 8)] scratch.
template <int V>
__device__ __forceinline__ void block_moments(const Running<V>& r, bool active, int lane, int col, int lanes, int C, int cg,
                                              float len, float* vals, float* red, float* s_mean, float* s_m2) {
  if (active) {
#pragma unroll
    for (int i = 0; i < V; ++i) vals[lane * C + col * V + i] = r.n * r.mean[i];
  }
  int parts = group_sums(vals, lanes, C, cg, red);
  for (int g = threadIdx.x; g < C / cg; g += kGnThreads) s_mean[g] = sum_parts(red, g, parts) / (len * cg);
  __syncthreads();
  if (active) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float d = r.mean[i] - s_mean[(col * V + i) / cg];
      vals[lane * C + col * V + i] = fmaf(r.n * d, d, r.m2[i]);
    }
  }
  parts = group_sums(vals, lanes, C, cg, red);
  for (int g = threadIdx.x; g < C / cg; g += kGnThreads) s_m2[g] = sum_parts(red, g, parts);
  __syncthreads();
}

struct GnArgs {
  const void *x, *dout, *w, *b;
  int64_t HW;
  int C, cg;           // channels, channels per group
  int slab;            // channels per resident block
  int span;            // positions per block
  int n0;              // first sample (streamed)
  float eps;
  void* out;           // out or dx
  float *mean, *rstd;  // [N, G]
  float* part;         // streamed: [N][chunks][G][2] moments or [N][chunks][2][C] sums
  float* sums;         // [N][2][C] totals of g and g xh
};

template <class T>
__device__ __forceinline__ uint4 ld_raw(const T* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }
template <class T>
__device__ __forceinline__ void as_floats(const uint4& u, float (&f)[Vec<T>::V]) { Vec<T>::load(reinterpret_cast<const T*>(&u), f); }

// Parameters of a thread's channels
template <class T>
struct Affine {
  static constexpr int V = Vec<T>::V;
  float w[V], b[V];
  __device__ __forceinline__ Affine(const GnArgs& a, int ch) {
    Vec<T>::load(static_cast<const T*>(a.w) + ch, w);
    Vec<T>::load(static_cast<const T*>(a.b) + ch, b);
  }
};

template <class T, int ACT>
__global__ void __launch_bounds__(kGnThreads) groupnorm_resident_kernel(const GnArgs a) {
  constexpr int V = Vec<T>::V;
  extern __shared__ __align__(16) float gsm[];
  const int cols = a.slab / V, lanes = kGnThreads / cols, G = a.slab / a.cg;
  const int col = threadIdx.x % cols, lane = threadIdx.x / cols;
  const bool active = lane < lanes;
  const int cl = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
  const int n = blockIdx.z, c0 = blockIdx.y * a.slab;
  const int64_t p0 = min(a.HW, static_cast<int64_t>(rank) * a.span), p1 = min(a.HW, p0 + a.span);
  uint4* keep = reinterpret_cast<uint4*>(gsm);                       // [span][cols]
  float* vals = gsm + static_cast<int64_t>(a.span) * cols * 4;       // [lanes][slab]
  float* red = vals + lanes * a.slab;                                // [max(G, 8)]
  float* s_mean = red + max(G, kGnWarps);                            // [G], m2 behind it
  const int64_t base = (static_cast<int64_t>(n) * a.HW + p0) * a.C + c0 + col * V;
  const T* x = static_cast<const T*>(a.x) + base;
  const int len = static_cast<int>(p1 - p0);
  Running<V> r;
  if (active) {
    for (int p = lane; p < len; p += lanes * kGnBatch) {
      float f[kGnBatch][V];
      uint4 u[kGnBatch];
      int k = 0;
#pragma unroll
      for (int j = 0; j < kGnBatch; ++j) {
        u[j] = make_uint4(0u, 0u, 0u, 0u);
        if (p + j * lanes < len) u[j] = ld_raw(x + static_cast<int64_t>(p + j * lanes) * a.C), k = j + 1;
      }
#pragma unroll
      for (int j = 0; j < kGnBatch; ++j) {
        if (p + j * lanes < len) keep[(p + j * lanes) * cols + col] = u[j];
        as_floats<T>(u[j], f[j]);
      }
      r.add(f, k);
    }
  }
  block_moments<V>(r, active, lane, col, lanes, a.slab, a.cg, static_cast<float>(max(len, 1)), vals, red, s_mean,
                   s_mean + G);
  if (cl > 1) cluster_sync_all();
  // the cluster's blocks, in rank order: the mean first, then the deviations from it
  float* s_out = vals;                                               // [G] mean, [G] rstd
  for (int g = threadIdx.x; g < G; g += kGnThreads) {
    const uint32_t at = smem_u32(s_mean + g);
    float mu = 0.f, m2 = 0.f;
    for (int i = 0; i < cl; ++i) {
      const float ni = static_cast<float>(min(a.HW, static_cast<int64_t>(i + 1) * a.span) - min(a.HW, static_cast<int64_t>(i) * a.span));
      mu = fmaf(ni, ld_dsmem(mapa_shared(at, i)), mu);
    }
    mu /= static_cast<float>(a.HW);
    for (int i = 0; i < cl; ++i) {
      const float ni = static_cast<float>(min(a.HW, static_cast<int64_t>(i + 1) * a.span) - min(a.HW, static_cast<int64_t>(i) * a.span));
      const float d = ld_dsmem(mapa_shared(at, i)) - mu;
      m2 += fmaf(ni * a.cg * d, d, ld_dsmem(mapa_shared(at + G * 4, i)));
    }
    const float rs = rsqrtf(m2 / (static_cast<float>(a.HW) * a.cg) + a.eps);
    s_out[g] = mu, s_out[G + g] = rs;
    if (rank == 0 && a.mean != nullptr) {
      const int64_t to = static_cast<int64_t>(n) * (a.C / a.cg) + c0 / a.cg + g;
      a.mean[to] = mu, a.rstd[to] = rs;
    }
  }
  if (cl > 1) cluster_sync_all(); else __syncthreads();
  if (!active) return;
  const Affine<T> pr(a, c0 + col * V);
  float mu[V], rs[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int g = (col * V + i) / a.cg;
    mu[i] = s_out[g], rs[i] = s_out[G + g];
  }
  T* out = static_cast<T*>(a.out) + base;
  for (int p = lane; p < len; p += lanes) {
    float f[V];
    as_floats<T>(keep[p * cols + col], f);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = act_value<ACT, Vec<T>::exact>(fmaf((f[i] - mu[i]) * rs[i], pr.w[i], pr.b[i]));
    Vec<T>::store(out + static_cast<int64_t>(p) * a.C, f);
  }
}

// Sums of g and g xh of a thread's channels -> vals [2][lanes][C] -> per-channel totals tot[2][C] of the block
__device__ __forceinline__ void channel_totals(const float* vals, int lanes, int C, float* tot) {
  __syncthreads();
  // 4 threads per entry; C is a multiple of 4, so a warp's 8 entries are all there or none is
  for (int e = threadIdx.x / 4; e < 2 * C; e += kGnThreads / 4) {
    float s = 0.f;
    for (int l = threadIdx.x % 4; l < lanes; l += 4) s += vals[(e / C * lanes + l) * C + e % C];
    s += __shfl_xor_sync(0xffffffffu, s, 1);
    s += __shfl_xor_sync(0xffffffffu, s, 2);
    if (threadIdx.x % 4 == 0) tot[e] = s;
  }
  __syncthreads();
}

template <class T, int ACT>
struct Grad {
  static constexpr int V = Vec<T>::V;
  float mu[V], rs[V];
  __device__ __forceinline__ Grad(const GnArgs& a, int n, int ch) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int64_t g = static_cast<int64_t>(n) * (a.C / a.cg) + (ch + i) / a.cg;
      mu[i] = __ldg(a.mean + g), rs[i] = __ldg(a.rstd + g);
    }
  }
  __device__ __forceinline__ void sums(const Affine<T>& pr, const uint4& xu, const uint4& du, float (&sg)[V], float (&sx)[V]) const {
    float f[V], d[V];
    as_floats<T>(xu, f);
    as_floats<T>(du, d);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float xh = (f[i] - mu[i]) * rs[i];
      const float g = d[i] * act_slope<ACT, Vec<T>::exact>(fmaf(xh, pr.w[i], pr.b[i]));
      sg[i] += g;
      sx[i] = fmaf(g, xh, sx[i]);
    }
  }
  __device__ __forceinline__ void dx(const Affine<T>& pr, const float (&m1)[V], const float (&m2)[V], const uint4& xu,
                                     const uint4& du, T* to) const {
    float f[V], d[V];
    as_floats<T>(xu, f);
    as_floats<T>(du, d);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float xh = (f[i] - mu[i]) * rs[i];
      const float gw = d[i] * act_slope<ACT, Vec<T>::exact>(fmaf(xh, pr.w[i], pr.b[i])) * pr.w[i];
      f[i] = rs[i] * (gw - m1[i] - xh * m2[i]);
    }
    Vec<T>::store(to, f);
  }
};

template <class T, int ACT>
__global__ void __launch_bounds__(kGnThreads) groupnorm_bwd_resident_kernel(const GnArgs a) {
  constexpr int V = Vec<T>::V;
  extern __shared__ __align__(16) float gsm[];
  const int cols = a.slab / V, lanes = kGnThreads / cols, G = a.slab / a.cg, S = a.slab;
  const int col = threadIdx.x % cols, lane = threadIdx.x / cols;
  const bool active = lane < lanes;
  const int cl = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
  const int n = blockIdx.z, c0 = blockIdx.y * S;
  const int64_t p0 = min(a.HW, static_cast<int64_t>(rank) * a.span), p1 = min(a.HW, p0 + a.span);
  uint4* keep = reinterpret_cast<uint4*>(gsm);                       // [2][span][cols]
  float* vals = gsm + 2 * static_cast<int64_t>(a.span) * cols * 4;   // [2][lanes][S]
  float* tot = vals + 2 * lanes * S;                                 // [2][S]
  const int64_t base = (static_cast<int64_t>(n) * a.HW + p0) * a.C + c0 + col * V;
  const int len = static_cast<int>(p1 - p0);
  const Affine<T> pr(a, c0 + col * V);
  const Grad<T, ACT> gr(a, n, c0 + col * V);
  if (active) {
    float sg[V], sx[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sg[i] = 0.f, sx[i] = 0.f;
    const T *x = static_cast<const T*>(a.x) + base, *d = static_cast<const T*>(a.dout) + base;
    for (int p = lane; p < len; p += lanes * 2) {
      const bool two = p + lanes < len;
      const int64_t o0 = static_cast<int64_t>(p) * a.C, o1 = static_cast<int64_t>(p + lanes) * a.C;
      uint4 x0 = ld_raw(x + o0), d0 = ld_raw(d + o0), x1, d1;
      if (two) x1 = ld_raw(x + o1), d1 = ld_raw(d + o1);
      keep[p * cols + col] = x0, keep[(a.span + p) * cols + col] = d0;
      gr.sums(pr, x0, d0, sg, sx);
      if (two) {
        keep[(p + lanes) * cols + col] = x1, keep[(a.span + p + lanes) * cols + col] = d1;
        gr.sums(pr, x1, d1, sg, sx);
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      vals[lane * S + col * V + i] = sg[i];
      vals[(lanes + lane) * S + col * V + i] = sx[i];
    }
  }
  channel_totals(vals, lanes, S, tot);
  if (cl > 1) cluster_sync_all();
  float* all = vals;                                                 // [2][S] sums over the cluster, then [2][G] means
  for (int e = threadIdx.x; e < 2 * S; e += kGnThreads) {
    float s = 0.f;
    for (int i = 0; i < cl; ++i) s += ld_dsmem(mapa_shared(smem_u32(tot + e), i));
    if (rank == 0) a.sums[(static_cast<int64_t>(n) * 2 + e / S) * a.C + c0 + e % S] = s;
    all[e] = s * static_cast<float>(static_cast<const T*>(a.w)[c0 + e % S]);
  }
  if (cl > 1) cluster_sync_all(); else __syncthreads();
  for (int e = threadIdx.x; e < 2 * G; e += kGnThreads) {
    float s = 0.f;
    for (int c = 0; c < a.cg; ++c) s += all[e / G * S + e % G * a.cg + c];
    all[2 * S + e] = s / (static_cast<float>(a.HW) * a.cg);
  }
  __syncthreads();
  if (!active) return;
  float m1[V], m2[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int g = (col * V + i) / a.cg;
    m1[i] = all[2 * S + g], m2[i] = all[2 * S + G + g];
  }
  T* dx = static_cast<T*>(a.out) + base;
  for (int p = lane; p < len; p += lanes)
    gr.dx(pr, m1, m2, keep[p * cols + col], keep[(a.span + p) * cols + col], dx + static_cast<int64_t>(p) * a.C);
}

// part[n][chunk][g] = mean, squared deviations of the group over the chunk's positions
template <class T>
__global__ void __launch_bounds__(kGnThreads, 4) groupnorm_moments_kernel(const GnArgs a) {
  constexpr int V = Vec<T>::V;
  extern __shared__ __align__(16) float gsm[];
  const int cols = a.C / V, lanes = kGnThreads / cols, G = a.C / a.cg;
  const int col = threadIdx.x % cols, lane = threadIdx.x / cols;
  const int n = a.n0 + blockIdx.y;
  const int64_t p0 = static_cast<int64_t>(blockIdx.x) * a.span, p1 = min(a.HW, p0 + a.span);
  float *vals = gsm, *red = vals + lanes * a.C, *s_mean = red + max(G, kGnWarps);
  Running<V> r;
  if (lane < lanes) {
    const T* x = static_cast<const T*>(a.x) + (static_cast<int64_t>(n) * a.HW + p0) * a.C + col * V;
    const int len = static_cast<int>(p1 - p0);
    for (int p = lane; p < len; p += lanes * kGnBatch) {
      float f[kGnBatch][V];
      uint4 u[kGnBatch];
      int k = 0;
#pragma unroll
      for (int j = 0; j < kGnBatch; ++j) {
        u[j] = make_uint4(0u, 0u, 0u, 0u);
        if (p + j * lanes < len) u[j] = ld_raw(x + static_cast<int64_t>(p + j * lanes) * a.C), k = j + 1;
      }
#pragma unroll
      for (int j = 0; j < kGnBatch; ++j) as_floats<T>(u[j], f[j]);
      r.add(f, k);
    }
  }
  block_moments<V>(r, lane < lanes, lane, col, lanes, a.C, a.cg, static_cast<float>(p1 - p0), vals, red, s_mean, s_mean + G);
  for (int g = threadIdx.x; g < G; g += kGnThreads) {
    float* to = a.part + ((static_cast<int64_t>(n) * gridDim.x + blockIdx.x) * G + g) * 2;
    to[0] = s_mean[g], to[1] = s_mean[G + g];
  }
}

// Every block joins its sample's chunks (a warp per group, the same order everywhere) and normalises its own.
template <class T, int ACT>
__global__ void __launch_bounds__(kGnThreads, 4) groupnorm_apply_kernel(const GnArgs a) {
  constexpr int V = Vec<T>::V;
  extern __shared__ __align__(16) float gsm[];  // [G] mean, [G] rstd
  const int n = a.n0 + blockIdx.y, chunks = gridDim.x, G = a.C / a.cg;
  const float* part = a.part + static_cast<int64_t>(n) * chunks * G * 2;
  const float total = static_cast<float>(a.HW) * a.cg;
  for (int g = threadIdx.x / 32; g < G; g += kGnWarps) {
    auto len = [&](int k) { return static_cast<float>(min(a.HW - static_cast<int64_t>(k) * a.span, static_cast<int64_t>(a.span))) * a.cg; };
    auto warp_sum = [](float s) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      return s;
    };
    float s = 0.f;
    for (int k = threadIdx.x % 32; k < chunks; k += 32) s = fmaf(len(k), __ldg(part + (k * G + g) * 2), s);
    const float mu = warp_sum(s) / total;
    s = 0.f;
    for (int k = threadIdx.x % 32; k < chunks; k += 32) {
      const float2 m = __ldg(reinterpret_cast<const float2*>(part + (k * G + g) * 2));
      s += fmaf(len(k) * (m.x - mu), m.x - mu, m.y);
    }
    const float rs = rsqrtf(warp_sum(s) / total + a.eps);
    if (threadIdx.x % 32 == 0) {
      gsm[g] = mu, gsm[G + g] = rs;
      if (blockIdx.x == 0 && a.mean != nullptr) a.mean[static_cast<int64_t>(n) * G + g] = mu, a.rstd[static_cast<int64_t>(n) * G + g] = rs;
    }
  }
  __syncthreads();
  const int cols = a.C / V, lanes = kGnThreads / cols;
  const int col = threadIdx.x % cols, lane = threadIdx.x / cols;
  if (lane >= lanes) return;
  const Affine<T> pr(a, col * V);
  float mu[V], rs[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int g = (col * V + i) / a.cg;
    mu[i] = gsm[g], rs[i] = gsm[G + g];
  }
  const int64_t p0 = static_cast<int64_t>(blockIdx.x) * a.span;
  const int len = static_cast<int>(min(a.HW, p0 + a.span) - p0);
  const int64_t base = (static_cast<int64_t>(n) * a.HW + p0) * a.C + col * V;
  const T* x = static_cast<const T*>(a.x) + base;
  T* out = static_cast<T*>(a.out) + base;
  auto one = [&](const uint4& u, int p) {
    float f[V];
    as_floats<T>(u, f);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = act_value<ACT, Vec<T>::exact>(fmaf((f[i] - mu[i]) * rs[i], pr.w[i], pr.b[i]));
    Vec<T>::store(out + static_cast<int64_t>(p) * a.C, f);
  };
  for (int p = lane; p < len; p += lanes * 2) {
    const bool two = p + lanes < len;
    const uint4 u0 = ld_raw(x + static_cast<int64_t>(p) * a.C);
    uint4 u1;
    if (two) u1 = ld_raw(x + static_cast<int64_t>(p + lanes) * a.C);
    one(u0, p);
    if (two) one(u1, p + lanes);
  }
}

// part[n][chunk][0 | 1][c] = sums over the chunk's positions of g and of g xh
template <class T, int ACT>
__global__ void __launch_bounds__(kGnThreads, 2) groupnorm_bwd_sums_kernel(const GnArgs a) {
  constexpr int V = Vec<T>::V;
  extern __shared__ __align__(16) float gsm[];  // [2][lanes][C], [2][C]
  const int cols = a.C / V, lanes = kGnThreads / cols;
  const int col = threadIdx.x % cols, lane = threadIdx.x / cols;
  const int n = a.n0 + blockIdx.y;
  const int64_t p0 = static_cast<int64_t>(blockIdx.x) * a.span;
  if (lane < lanes) {
    const int len = static_cast<int>(min(a.HW, p0 + a.span) - p0);
    const Affine<T> pr(a, col * V);
    const Grad<T, ACT> gr(a, n, col * V);
    float sg[V], sx[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sg[i] = 0.f, sx[i] = 0.f;
    const int64_t base = (static_cast<int64_t>(n) * a.HW + p0) * a.C + col * V;
    const T *x = static_cast<const T*>(a.x) + base, *d = static_cast<const T*>(a.dout) + base;
    for (int p = lane; p < len; p += lanes * 2) {
      const bool two = p + lanes < len;
      const int64_t o0 = static_cast<int64_t>(p) * a.C, o1 = static_cast<int64_t>(p + lanes) * a.C;
      const uint4 x0 = ld_raw(x + o0), d0 = ld_raw(d + o0);
      uint4 x1, d1;
      if (two) x1 = ld_raw(x + o1), d1 = ld_raw(d + o1);
      gr.sums(pr, x0, d0, sg, sx);
      if (two) gr.sums(pr, x1, d1, sg, sx);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      gsm[lane * a.C + col * V + i] = sg[i];
      gsm[(lanes + lane) * a.C + col * V + i] = sx[i];
    }
  }
  float* tot = gsm + 2 * lanes * a.C;
  channel_totals(gsm, lanes, a.C, tot);
  float* to = a.part + (static_cast<int64_t>(n) * gridDim.x + blockIdx.x) * 2 * a.C;
  for (int e = threadIdx.x; e < 2 * a.C; e += kGnThreads) to[e] = tot[e];
}

// sums[n][..] = the sample's chunks; a warp's lanes are 32 entries, its block's warps share the chunks
__global__ void __launch_bounds__(1024) groupnorm_bwd_totals_kernel(const float* part, int n0, int chunks, int C, float* sums) {
  __shared__ float sm[32][33];
  const int n = n0 + blockIdx.y, e = blockIdx.x * 32 + threadIdx.x;
  float s = 0.f;
  if (e < 2 * C)
    for (int k = threadIdx.y; k < chunks; k += 32) s += part[(static_cast<int64_t>(n) * chunks + k) * 2 * C + e];
  sm[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  s = sm[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int to = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && to < 2 * C) sums[static_cast<int64_t>(n) * 2 * C + to] = s;
}

template <class T, int ACT>
__global__ void __launch_bounds__(kGnThreads, 2) groupnorm_bwd_dx_kernel(const GnArgs a) {
  constexpr int V = Vec<T>::V;
  extern __shared__ __align__(16) float gsm[];  // [2][C] sums times w, [2][G] group means
  const int n = a.n0 + blockIdx.y, G = a.C / a.cg;
  for (int c = threadIdx.x; c < 2 * a.C; c += kGnThreads)
    gsm[c] = a.sums[static_cast<int64_t>(n) * 2 * a.C + c] * static_cast<float>(static_cast<const T*>(a.w)[c % a.C]);
  __syncthreads();
  for (int e = threadIdx.x; e < 2 * G; e += kGnThreads) {
    float s = 0.f;
    for (int c = 0; c < a.cg; ++c) s += gsm[e / G * a.C + e % G * a.cg + c];
    gsm[2 * a.C + e] = s / (static_cast<float>(a.HW) * a.cg);
  }
  __syncthreads();
  const int cols = a.C / V, lanes = kGnThreads / cols;
  const int col = threadIdx.x % cols, lane = threadIdx.x / cols;
  if (lane >= lanes) return;
  const Affine<T> pr(a, col * V);
  const Grad<T, ACT> gr(a, n, col * V);
  float m1[V], m2[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int g = (col * V + i) / a.cg;
    m1[i] = gsm[2 * a.C + g], m2[i] = gsm[2 * a.C + G + g];
  }
  const int64_t p0 = static_cast<int64_t>(blockIdx.x) * a.span;
  const int len = static_cast<int>(min(a.HW, p0 + a.span) - p0);
  const int64_t base = (static_cast<int64_t>(n) * a.HW + p0) * a.C + col * V;
  const T *x = static_cast<const T*>(a.x) + base, *d = static_cast<const T*>(a.dout) + base;
  T* dx = static_cast<T*>(a.out) + base;
  for (int p = lane; p < len; p += lanes * 2) {
    const bool two = p + lanes < len;
    const int64_t o0 = static_cast<int64_t>(p) * a.C, o1 = static_cast<int64_t>(p + lanes) * a.C;
    const uint4 x0 = ld_raw(x + o0), d0 = ld_raw(d + o0);
    uint4 x1, d1;
    if (two) x1 = ld_raw(x + o1), d1 = ld_raw(d + o1);
    gr.dx(pr, m1, m2, x0, d0, dx + o0);
    if (two) gr.dx(pr, m1, m2, x1, d1, dx + o1);
  }
}

// db[c] = sum over the P partials of sums[p][0][c], dw[c] of sums[p][1][c]
template <class T>
__global__ void __launch_bounds__(1024) norm_param_grad_kernel(const float* __restrict__ sums, int P, int C,
                                                               T* __restrict__ dw, T* __restrict__ db) {
  __shared__ float sm[32][33];
  const int e = blockIdx.x * 32 + threadIdx.x;
  float s = 0.f;
  if (e < 2 * C) {
#pragma unroll 4
    for (int p = threadIdx.y; p < P; p += 32) s += sums[static_cast<int64_t>(p) * 2 * C + e];
  }
  sm[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  s = sm[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int to = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && to < 2 * C) norm_store1(to < C ? db + to : dw + (to - C), s);
}

static size_t gn_align(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }

// How a call is cut up (see the top of this part).
struct GnPlan {
  int slab, cluster, span;     // resident; cluster 0: streamed
  int batch, chunks;           // streamed: samples per launch, blocks per sample
  size_t smem;
};

static size_t gn_resident_smem(int64_t span, int slab, int cg, int elem, bool backward) {
  const int V = 16 / elem, lanes = kGnThreads / (slab / V), G = slab / cg;
  const size_t keep = static_cast<size_t>(span) * slab * elem * (backward ? 2 : 1);
  return backward ? keep + (2 * static_cast<size_t>(lanes) * slab + 2 * slab) * 4
                  : keep + (static_cast<size_t>(lanes) * slab + std::max(G, kGnWarps) + 2 * G) * 4;
}

static GnPlan groupnorm_plan(int N, int64_t HW, int C, int groups, int elem, bool backward) {
  GnPlan p = {};
  const int V = 16 / elem, cg = C / groups;
  // the narrowest slab of whole groups and whole vectors that is at least 64 bytes wide and divides C
  int slab = C;
  for (int k = 1; k <= groups; ++k)
    if (groups % k == 0 && k * cg % V == 0 && k * cg * elem >= 64) {
      slab = k * cg;
      break;
    }
  // scratch of the backward's [2][S] + [2][G] totals lies in the lanes' [2][lanes][S]
  const bool room = kGnThreads / (slab / V) >= 2;
  int cl = 1;
  const int64_t clusters = static_cast<int64_t>(N) * (C / slab);
  while (cl < 8 && HW > cl * 64 &&
         (clusters * cl < 148 || gn_resident_smem((HW + cl - 1) / cl, slab, cg, elem, backward) > kGnResident / 2))
    cl *= 2;
  const int64_t span = (HW + cl - 1) / cl;
  if (room && span < (1 << 20) && gn_resident_smem(span, slab, cg, elem, backward) <= static_cast<size_t>(kGnResident)) {
    p.slab = slab, p.cluster = cl, p.span = static_cast<int>(span);
    p.smem = gn_resident_smem(span, slab, cg, elem, backward);
    return p;
  }
  const int64_t sample = HW * C * elem * (backward ? 2 : 1);
  p.batch = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(N, kGnL2 / sample)));
  const int per_sm = backward ? 2 : 4;
  const int64_t want = std::max<int64_t>(1, (148 * per_sm + p.batch - 1) / p.batch);
  p.span = static_cast<int>(std::max<int64_t>(32, (HW + want - 1) / want));
  p.chunks = static_cast<int>((HW + p.span - 1) / p.span);
  return p;
}

size_t groupnorm_workspace_size(int N, int64_t HW, int C, int groups, int dtype, int backward) {
  if (N <= 0 || HW <= 0 || C <= 0 || groups <= 0 || C % groups || dtype < 0 || dtype > 2) return 0;
  const GnPlan p = groupnorm_plan(N, HW, C, groups, dtype == 2 ? 4 : 2, backward != 0);
  const size_t part = p.cluster ? 0 : static_cast<size_t>(N) * p.chunks * 2 * (backward ? C : groups) * sizeof(float);
  const size_t sums = backward ? static_cast<size_t>(N) * 2 * C * sizeof(float) : 0;
  return gn_align(part) + gn_align(sums);
}

static int groupnorm_check(int N, int64_t HW, int C, int G, int act, int dtype, size_t workspace_bytes,
                           const void* workspace, int backward) {
  if (N <= 0 || HW <= 0 || C <= 0 || G <= 0 || C % G || act < 0 || act > 3 || dtype < 0 || dtype > 2)
    return SSAM_ERR_INVALID;
  const int V = dtype == 2 ? 4 : 8;
  if (C % V || C / V > kGnThreads || N > 65535 || HW > (1ll << 31)) return SSAM_ERR_UNSUPPORTED;
  const size_t need = groupnorm_workspace_size(N, HW, C, G, dtype, backward);
  if (workspace_bytes < need || (need > 0 && workspace == nullptr)) return SSAM_ERR_INVALID;
  return SSAM_OK;
}

template <class K>
static int launch_gn_cluster(K kernel, PerDeviceOnce& once, dim3 grid, size_t smem, int cluster, cudaStream_t stream,
                             const GnArgs& a) {
  const int st = once.run(current_device(), [&] {
    return status_from_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 static_cast<int>(kGnResident)));
  });
  if (st != SSAM_OK) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kGnThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return status_from_cuda(cudaLaunchKernelEx(&cfg, kernel, a));
}

template <class T, int ACT>
static int groupnorm_fwd_t(GnArgs a, int N, int G, float* ws, cudaStream_t stream) {
  static PerDeviceOnce once;
  const GnPlan p = groupnorm_plan(N, a.HW, a.C, G, sizeof(T), false);
  a.span = p.span, a.slab = p.slab, a.part = ws;
  if (p.cluster)
    return launch_gn_cluster(groupnorm_resident_kernel<T, ACT>, once, dim3(p.cluster, a.C / p.slab, N), p.smem, p.cluster,
                             stream, a);
  const int lanes = kGnThreads / (a.C / Vec<T>::V);
  for (a.n0 = 0; a.n0 < N; a.n0 += p.batch) {
    const dim3 grid(p.chunks, std::min(p.batch, N - a.n0));
    groupnorm_moments_kernel<T><<<grid, kGnThreads, (lanes * a.C + std::max(G, kGnWarps) + 2 * G) * sizeof(float), stream>>>(a);
    groupnorm_apply_kernel<T, ACT><<<grid, kGnThreads, 2 * G * sizeof(float), stream>>>(a);
    const int st = status_from_cuda(cudaGetLastError());
    if (st != SSAM_OK) return st;
  }
  return SSAM_OK;
}

template <class T, int ACT>
static int groupnorm_bwd_t(GnArgs a, int N, int G, void* dw, void* db, float* ws, cudaStream_t stream) {
  static PerDeviceOnce once;
  const GnPlan p = groupnorm_plan(N, a.HW, a.C, G, sizeof(T), true);
  a.span = p.span, a.slab = p.slab, a.sums = ws;
  a.part = ws + gn_align(static_cast<size_t>(N) * 2 * a.C * sizeof(float)) / sizeof(float);
  int st;
  if (p.cluster) {
    st = launch_gn_cluster(groupnorm_bwd_resident_kernel<T, ACT>, once, dim3(p.cluster, a.C / p.slab, N), p.smem, p.cluster,
                           stream, a);
    if (st != SSAM_OK) return st;
  } else {
    const int lanes = kGnThreads / (a.C / Vec<T>::V);
    for (a.n0 = 0; a.n0 < N; a.n0 += p.batch) {
      const dim3 grid(p.chunks, std::min(p.batch, N - a.n0));
      groupnorm_bwd_sums_kernel<T, ACT><<<grid, kGnThreads, (2 * lanes * a.C + 2 * a.C) * sizeof(float), stream>>>(a);
      groupnorm_bwd_totals_kernel<<<dim3((2 * a.C + 31) / 32, grid.y), dim3(32, 32), 0, stream>>>(a.part, a.n0, p.chunks, a.C, a.sums);
      groupnorm_bwd_dx_kernel<T, ACT><<<grid, kGnThreads, 2 * static_cast<size_t>(a.C + G) * sizeof(float), stream>>>(a);
      st = status_from_cuda(cudaGetLastError());
      if (st != SSAM_OK) return st;
    }
  }
  norm_param_grad_kernel<T><<<(2 * a.C + 31) / 32, dim3(32, 32), 0, stream>>>(a.sums, N, a.C, static_cast<T*>(dw), static_cast<T*>(db));
  return status_from_cuda(cudaGetLastError());
}

#define SSAM_GN_ACT(T, call)                         \
  switch (act) {                                     \
    case kActNone: return call<T, kActNone> ARGS;    \
    case kActRelu: return call<T, kActRelu> ARGS;    \
    case kActGelu: return call<T, kActGelu> ARGS;    \
    default: return call<T, kActSilu> ARGS;          \
  }

int groupnorm_act_fwd(const void* x, int N, int64_t HW, int C, int groups, const void* w, const void* b, float eps,
                      int act, int dtype, void* out, float* mean, float* rstd, void* workspace, size_t workspace_bytes,
                      cudaStream_t stream) {
  if (x == nullptr || w == nullptr || b == nullptr || out == nullptr || (mean == nullptr) != (rstd == nullptr))
    return SSAM_ERR_INVALID;
  const int st = groupnorm_check(N, HW, C, groups, act, dtype, workspace_bytes, workspace, 0);
  if (st != SSAM_OK) return st;
  for (const void* p : {x, w, b, static_cast<const void*>(out), static_cast<const void*>(workspace)})
    if (!aligned16(p)) return SSAM_ERR_ALIGN;
  GnArgs a = {};
  a.x = x, a.w = w, a.b = b, a.HW = HW, a.C = C, a.cg = C / groups, a.eps = eps, a.out = out, a.mean = mean, a.rstd = rstd;
  float* ws = static_cast<float*>(workspace);
#define ARGS (a, N, groups, ws, stream)
  if (dtype == 0) SSAM_GN_ACT(__half, groupnorm_fwd_t)
  if (dtype == 1) SSAM_GN_ACT(__nv_bfloat16, groupnorm_fwd_t)
  SSAM_GN_ACT(float, groupnorm_fwd_t)
#undef ARGS
}

int groupnorm_act_bwd(const void* x, const void* dout, int N, int64_t HW, int C, int groups, const void* w,
                      const void* b, const float* mean, const float* rstd, int act, int dtype, void* dx, void* dw,
                      void* db, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  if (x == nullptr || dout == nullptr || w == nullptr || b == nullptr || mean == nullptr || rstd == nullptr ||
      dx == nullptr || dw == nullptr || db == nullptr)
    return SSAM_ERR_INVALID;
  const int st = groupnorm_check(N, HW, C, groups, act, dtype, workspace_bytes, workspace, 1);
  if (st != SSAM_OK) return st;
  for (const void* p : {x, dout, w, b, static_cast<const void*>(dx), static_cast<const void*>(workspace)})
    if (!aligned16(p)) return SSAM_ERR_ALIGN;
  GnArgs a = {};
  a.x = x, a.dout = dout, a.w = w, a.b = b, a.HW = HW, a.C = C, a.cg = C / groups, a.out = dx;
  a.mean = const_cast<float*>(mean), a.rstd = const_cast<float*>(rstd);
  float* ws = static_cast<float*>(workspace);
#define ARGS (a, N, groups, dw, db, ws, stream)
  if (dtype == 0) SSAM_GN_ACT(__half, groupnorm_bwd_t)
  if (dtype == 1) SSAM_GN_ACT(__nv_bfloat16, groupnorm_bwd_t)
  SSAM_GN_ACT(float, groupnorm_bwd_t)
#undef ARGS
}

// ---------------------------------------------------------------------------
// Backward of ssam_layernorm_gelu_half: C / 8 threads per row, as the forward;
// the row's moments are recomputed from x (it is read anyway). Each block sums its
// rows' parameter gradients into one partial.
// ---------------------------------------------------------------------------
template <class T, int C, bool GELU>
__global__ void __launch_bounds__(256) layernorm_half_bwd_kernel(const T* __restrict__ x, const T* __restrict__ dout,
                                                                 int64_t rows, const T* __restrict__ w,
                                                                 const T* __restrict__ b, float eps, T* __restrict__ dx,
                                                                 float* __restrict__ sums) {
  constexpr int TPR = C / 8, RPB = 256 / TPR;
  __shared__ float part[RPB][2][C];
  const int t = threadIdx.x % TPR, lr = threadIdx.x / TPR;
  float wf[8], bf[8], sg[8], sx[8];
  Vec<T>::load(w + t * 8, wf);
  Vec<T>::load(b + t * 8, bf);
#pragma unroll
  for (int i = 0; i < 8; ++i) sg[i] = 0.f, sx[i] = 0.f;
  auto row_sum = [](float v) {
#pragma unroll
    for (int o = 1; o < TPR; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * RPB; r0 < rows; r0 += static_cast<int64_t>(gridDim.x) * RPB) {
    const int64_t r = r0 + lr;
    const bool ok = r < rows;
    float f[8], d[8];
    if (ok) {
      Vec<T>::load(x + r * C + t * 8, f);
      Vec<T>::load(dout + r * C + t * 8, d);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = 0.f, d[i] = 0.f;
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += f[i];
    const float mu = row_sum(s) * (1.f / C);
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] -= mu, s = fmaf(f[i], f[i], s);
    const float rs = rsqrtf(row_sum(s) * (1.f / C) + eps);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f[i] *= rs;
      const float g = GELU ? d[i] * act_slope<kActGelu, false>(fmaf(f[i], wf[i], bf[i])) : d[i];
      sg[i] += g;
      sx[i] = fmaf(g, f[i], sx[i]);
      d[i] = g * wf[i];
      s1 += d[i];
      s2 = fmaf(d[i], f[i], s2);
    }
    s1 = row_sum(s1) * (1.f / C);
    s2 = row_sum(s2) * (1.f / C);
    if (ok) {
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] = rs * (d[i] - s1 - f[i] * s2);
      Vec<T>::store(dx + r * C + t * 8, d);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) part[lr][0][t * 8 + i] = sg[i], part[lr][1][t * 8 + i] = sx[i];
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * C; c += 256) {
    float s = 0.f;
    for (int k = 0; k < RPB; ++k) s += part[k][c / C][c % C];
    sums[static_cast<int64_t>(blockIdx.x) * 2 * C + c] = s;
  }
}

static int layernorm_bwd_blocks(int64_t rows, int C) {
  const int64_t per = 256 / (C / 8);
  return static_cast<int>(std::min<int64_t>((rows + per - 1) / per, 4 * 148));
}

size_t layernorm_half_bwd_workspace_size(int64_t rows, int C) {
  if (rows <= 0 || C < 32 || C > 256) return 0;
  return gn_align(static_cast<size_t>(layernorm_bwd_blocks(rows, C)) * 2 * C * sizeof(float));
}

template <class T, int C>
static int layernorm_half_bwd_c(const void* x, const void* dout, int64_t rows, const void* w, const void* b, float eps,
                                int gelu, void* dx, void* dw, void* db, float* ws, cudaStream_t stream) {
  const int blocks = layernorm_bwd_blocks(rows, C);
  auto* kernel = gelu ? layernorm_half_bwd_kernel<T, C, true> : layernorm_half_bwd_kernel<T, C, false>;
  kernel<<<blocks, 256, 0, stream>>>(static_cast<const T*>(x), static_cast<const T*>(dout), rows,
                                     static_cast<const T*>(w), static_cast<const T*>(b), eps, static_cast<T*>(dx), ws);
  const int st = status_from_cuda(cudaGetLastError());
  if (st != SSAM_OK) return st;
  norm_param_grad_kernel<T><<<(2 * C + 31) / 32, dim3(32, 32), 0, stream>>>(ws, blocks, C, static_cast<T*>(dw),
                                                                           static_cast<T*>(db));
  return status_from_cuda(cudaGetLastError());
}

template <class T>
static int layernorm_half_bwd_t(const void* x, const void* dout, int64_t rows, int C, const void* w, const void* b,
                                float eps, int gelu, void* dx, void* dw, void* db, float* ws, cudaStream_t stream) {
  switch (C) {
    case 32: return layernorm_half_bwd_c<T, 32>(x, dout, rows, w, b, eps, gelu, dx, dw, db, ws, stream);
    case 64: return layernorm_half_bwd_c<T, 64>(x, dout, rows, w, b, eps, gelu, dx, dw, db, ws, stream);
    case 128: return layernorm_half_bwd_c<T, 128>(x, dout, rows, w, b, eps, gelu, dx, dw, db, ws, stream);
    case 256: return layernorm_half_bwd_c<T, 256>(x, dout, rows, w, b, eps, gelu, dx, dw, db, ws, stream);
    default: return SSAM_ERR_UNSUPPORTED;
  }
}

int layernorm_half_bwd(const void* x, const void* dout, int64_t rows, int C, const void* w, const void* b, float eps,
                       int gelu, int dtype, void* dx, void* dw, void* db, void* workspace, size_t workspace_bytes,
                       cudaStream_t stream) {
  if (x == nullptr || dout == nullptr || w == nullptr || b == nullptr || dx == nullptr || dw == nullptr ||
      db == nullptr || rows <= 0 || dtype < 0 || dtype > 1 || gelu < 0 || gelu > 1)
    return SSAM_ERR_INVALID;
  if (C != 32 && C != 64 && C != 128 && C != 256) return SSAM_ERR_UNSUPPORTED;
  if (workspace == nullptr || workspace_bytes < layernorm_half_bwd_workspace_size(rows, C)) return SSAM_ERR_INVALID;
  for (const void* p : {x, dout, w, b, static_cast<const void*>(dx), static_cast<const void*>(workspace)})
    if (!aligned16(p)) return SSAM_ERR_ALIGN;
  float* ws = static_cast<float*>(workspace);
  if (dtype == 0) return layernorm_half_bwd_t<__half>(x, dout, rows, C, w, b, eps, gelu, dx, dw, db, ws, stream);
  return layernorm_half_bwd_t<__nv_bfloat16>(x, dout, rows, C, w, b, eps, gelu, dx, dw, db, ws, stream);
}

}  // namespace ssam
