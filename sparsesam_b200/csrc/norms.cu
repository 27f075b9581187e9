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

#define SSAM_NO_WAITS
#include "common.cuh"
#include "host_util.h"

namespace ssam {

enum { kActNone = 0, kActRelu = 1, kActGelu = 2, kActSilu = 3 };

// act(z) and act'(z). EXACT (fp32 maps) takes the full-precision functions. The half
// types take erf from Abramowitz & Stegun 7.1.26 (as gelu_exact, |error| 1.5e-7; the
// exponential of erf is the one of GELU's slope) and the approximate exponential and
// division: a thousandth of the output's rounding, and 2 to 3 times fewer instructions,
// which is what bounded these kernels (GELU apply of 16 x 256 x 256 x 64: 108 us exact).
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
// 1 / (1 + p u) of a pair from one reciprocal of the product (both factors are 1 to 6.3, see erf_terms2): the
// reciprocals and exponentials (MUFU, a quarter of the FMA rate) are what GELU waits for.
__device__ __forceinline__ float2 erf_t2(float2 u) {
  const float2 d = fma2(both(0.3275911f), u, both(1.0f));
  const float r = rcp_fast(d.x * d.y);
  return mul2(both(r), make_float2(d.y, d.x));
}
// h = q / 2 of 7.1.26 without its exponential, e = exp(-u^2). u goes no further than 16, where e is 0 (2^-369): what
// meets e stays finite, and of two channels one that is not finite leaves the other's reciprocal alone (NaN comes
// through e, from the u that was not cut).
__device__ __forceinline__ void erf_terms2(float2 z, float2& u, float2& h, float2& e) {
  u = mul2(make_float2(fabsf(z.x), fabsf(z.y)), both(0.70710678118654752440f));
  const float2 arg = mul2(mul2(u, u), both(-1.4426950408889634f));
  e = make_float2(ex2f(arg.x), ex2f(arg.y));
  u = make_float2(fminf(u.x, 16.f), fminf(u.y, 16.f));
  const float2 t = erf_t2(u);
  h = fma2(both(0.5307027145f), t, both(-0.7265760135f));
  h = fma2(h, t, both(0.7107068705f));
  h = fma2(h, t, both(-0.142248368f));
  h = fma2(h, t, both(0.127414796f));
  h = mul2(h, t);
}
// GELU(z) = max(z, 0) - |z| h e
__device__ __forceinline__ float2 gelu2(float2 z) {
  float2 u, h, e;
  erf_terms2(z, u, h, e);
  return fma2(mul2(u, both(-1.41421356237309504880f)), mul2(h, e), make_float2(fmaxf(z.x, 0.f), fmaxf(z.y, 0.f)));
}
// GELU'(z) = Phi(z) + z phi(z), Phi = 1/2 + sign(z) (1/2 - h e)
__device__ __forceinline__ float2 gelu_slope2(float2 z) {
  float2 u, h, e;
  erf_terms2(z, u, h, e);
  const float2 half = fma2(h, make_float2(-e.x, -e.y), both(0.5f));
  const float2 phi = make_float2(copysignf(half.x, z.x), copysignf(half.y, z.y));
  return add2(fma2(mul2(z, both(0.39894228040143267794f)), e, phi), both(0.5f));
}
template <int ACT, bool EXACT>
__device__ __forceinline__ float2 act_value(float2 z) {
  if constexpr (ACT == kActRelu) return make_float2(z.x < 0.f ? 0.f : z.x, z.y < 0.f ? 0.f : z.y);  // NaN stays NaN
  if constexpr (ACT == kActGelu) {
    if constexpr (!EXACT) return gelu2(z);
    return make_float2(0.5f * z.x * (1.f + erff(z.x * 0.70710678118654752440f)),
                       0.5f * z.y * (1.f + erff(z.y * 0.70710678118654752440f)));
  }
  if constexpr (ACT == kActSilu) {
    if constexpr (EXACT) return make_float2(z.x / (1.f + expf(-z.x)), z.y / (1.f + expf(-z.y)));
    return make_float2(__fdividef(z.x, 1.f + __expf(-z.x)), __fdividef(z.y, 1.f + __expf(-z.y)));
  }
  return z;
}
template <bool EXACT>
__device__ __forceinline__ float silu_slope(float z) {
  const float s = EXACT ? 1.f / (1.f + expf(-z)) : rcp_fast(1.f + __expf(-z));
  return s * (1.f + z * (1.f - s));
}
__device__ __forceinline__ float gelu_slope_exact(float z) {
  return 0.5f * (1.f + erff(z * 0.70710678118654752440f)) + z * expf(-0.5f * z * z) * 0.39894228040143267794f;
}
template <int ACT, bool EXACT>
__device__ __forceinline__ float2 act_slope(float2 z) {
  if constexpr (ACT == kActRelu) return make_float2(z.x > 0.f ? 1.f : 0.f, z.y > 0.f ? 1.f : 0.f);
  if constexpr (ACT == kActGelu) {
    if constexpr (EXACT) return make_float2(gelu_slope_exact(z.x), gelu_slope_exact(z.y));
    return gelu_slope2(z);
  }
  if constexpr (ACT == kActSilu) return make_float2(silu_slope<EXACT>(z.x), silu_slope<EXACT>(z.y));
  return both(1.f);
}

// V consecutive channels (16 bytes) of a row as V / 2 pairs of floats.
template <class T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int V = 4;
  static constexpr bool exact = true;
  static __device__ __forceinline__ void unpack(const uint4& u, float2 (&f)[2]) {
    f[0] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
    f[1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&f)[2]) {
    return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x), __float_as_uint(f[1].y));
  }
};
template <>
struct Vec<__half> {
  static constexpr int V = 8;
  static constexpr bool exact = false;
  static __device__ __forceinline__ void unpack(const uint4& u, float2 (&f)[4]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&f)[4]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(f[i].x, f[i].y);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int V = 8;
  static constexpr bool exact = false;
  static __device__ __forceinline__ void unpack(const uint4& u, float2 (&f)[4]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&f)[4]) {
    return make_uint4(pack_bf16x2(f[0].x, f[0].y), pack_bf16x2(f[1].x, f[1].y), pack_bf16x2(f[2].x, f[2].y),
                      pack_bf16x2(f[3].x, f[3].y));
  }
};
template <class T>
__device__ __forceinline__ uint4 ld_raw(const T* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }
template <class T>
__device__ __forceinline__ void st_raw(T* p, const uint4& u) { *reinterpret_cast<uint4*>(p) = u; }
template <class T>
__device__ __forceinline__ void load_pairs(const T* p, float2 (&f)[Vec<T>::V / 2]) { Vec<T>::unpack(ld_raw(p), f); }

// A thread's private ring of D slots of S 16-byte vectors in shared memory, filled by cp.async: loads stay in
// flight under the arithmetic without holding registers. Nothing is shared between threads, so a thread waits
// for its own copies only.
template <int D, int S, int THREADS>
struct Ring {
  uint32_t base;
  __device__ __forceinline__ explicit Ring(const void* smem) : base(smem_u32(smem) + threadIdx.x * 16) {}
  static constexpr int bytes = D * S * THREADS * 16;
  __device__ __forceinline__ void fetch(int slot, int s, const void* src) const {
    cp_async16(base + (slot * S + s) * THREADS * 16, src, 16);
  }
  static __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
  static __device__ __forceinline__ void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(D - 1) : "memory"); }
  __device__ __forceinline__ uint4 get(int slot, int s) const {
    uint4 u;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                 : "r"(base + (slot * S + s) * THREADS * 16)
                 : "memory");
    return u;
  }
  // body(p, raw0[, raw1]) for p = first, first + step, .. < len; vector s of position p is at src_s + p * stride
  template <class T, class B>
  __device__ __forceinline__ void walk(const T* src0, const T* src1, int first, int step, int len, int stride, B body) const {
    auto request = [&](int slot, int p) {
      if (p < len) {
        fetch(slot, 0, src0 + static_cast<int64_t>(p) * stride);
        if (S == 2) fetch(slot, 1, src1 + static_cast<int64_t>(p) * stride);
      }
      commit();
    };
#pragma unroll
    for (int i = 0; i < D; ++i) request(i, first + i * step);
    for (int p = first; p < len; p += D * step) {
#pragma unroll
      for (int i = 0; i < D; ++i) {
        const int at = p + i * step;
        if (at >= len) break;
        wait();
        const uint4 u0 = get(i, 0);
        body(at, u0, S == 2 ? get(i, 1) : u0);
        request(i, at + D * step);           // the slot's values have been used
      }
    }
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
//    launched for as many samples at a time as stay in L2 between the two (72 MB; 48 MB
//    measured 301 us, 72 MB 274, 100 MB 280 on 16 x 256 x 256 x 64 bf16 GELU with gradients),
//    so that HBM still sees x about once.
// ---------------------------------------------------------------------------
constexpr int kGnThreads = 256;
constexpr int kGnWarps = kGnThreads / 32;
constexpr int kGnBatch = 4;                     // positions loaded ahead; their moments are exact, then merged
constexpr int64_t kGnResident = 96 << 10;       // shared-memory bytes a resident block may hold (two blocks per SM)
constexpr int64_t kGnL2 = 72 << 20;             // bytes of a streamed batch of samples

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
  static constexpr int P = V / 2;
  float n = 0.f;
  float2 mean[P], m2[P];
  __device__ __forceinline__ Running() {
#pragma unroll
    for (int i = 0; i < P; ++i) mean[i] = m2[i] = both(0.f);
  }
  template <int K>
  __device__ __forceinline__ void add(const float2 (&f)[K][P]) {
    const float nn = n + K, w = __fdividef(static_cast<float>(K), nn), cw = n * w;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      float2 s = f[0][i], q = both(0.f);
#pragma unroll
      for (int j = 1; j < K; ++j) s = add2(s, f[j][i]);
      if (K > 1) {
        s = mul2(s, both(-1.f / K));
#pragma unroll
        for (int j = 0; j < K; ++j) {
          const float2 d = add2(f[j][i], s);
          q = fma2(d, d, q);
        }
        s = mul2(s, both(-1.f));
      }
      const float2 d = fma2(mean[i], both(-1.f), s);
      mean[i] = fma2(d, both(w), mean[i]);
      m2[i] = add2(m2[i], fma2(mul2(d, d), both(cw), q));
    }
    n = nn;
  }
  // positions lane, lane + lanes, .. < len of x (stride C); keep(p, raw) sees each of them
  template <class T, class Keep>
  __device__ __forceinline__ void walk(const T* x, int lane, int lanes, int len, int C, Keep keep) {
    int p = lane;
    for (; p + (kGnBatch - 1) * lanes < len; p += lanes * kGnBatch) {
      uint4 u[kGnBatch];
      float2 f[kGnBatch][P];
#pragma unroll
      for (int j = 0; j < kGnBatch; ++j) u[j] = ld_raw(x + static_cast<int64_t>(p + j * lanes) * C);
#pragma unroll
      for (int j = 0; j < kGnBatch; ++j) {
        keep(p + j * lanes, u[j]);
        Vec<T>::unpack(u[j], f[j]);
      }
      add(f);
    }
    uint4 u[kGnBatch - 1];
#pragma unroll
    for (int j = 0; j < kGnBatch - 1; ++j)
      if (p + j * lanes < len) u[j] = ld_raw(x + static_cast<int64_t>(p + j * lanes) * C);
#pragma unroll
    for (int j = 0; j < kGnBatch - 1; ++j)
      if (p + j * lanes < len) {
        float2 f[1][P];
        keep(p + j * lanes, u[j]);
        Vec<T>::unpack(u[j], f[0]);
        add(f);
      }
  }
};

// Group means and squared deviations of a block's positions [len] from the threads' running moments:
// s_mean[g], s_m2[g]. vals: [lanes][C], red: [max(G, 8)] scratch.
template <int V>
__device__ __forceinline__ void block_moments(const Running<V>& r, bool active, int lane, int col, int lanes, int C, int cg,
                                              float len, float* vals, float* red, float* s_mean, float* s_m2) {
  if (active) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      vals[lane * C + col * V + 2 * i] = r.n * r.mean[i].x;
      vals[lane * C + col * V + 2 * i + 1] = r.n * r.mean[i].y;
    }
  }
  int parts = group_sums(vals, lanes, C, cg, red);
  for (int g = threadIdx.x; g < C / cg; g += kGnThreads) s_mean[g] = sum_parts(red, g, parts) / (len * cg);
  __syncthreads();
  if (active) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float d = (i & 1 ? r.mean[i / 2].y : r.mean[i / 2].x) - s_mean[(col * V + i) / cg];
      vals[lane * C + col * V + i] = fmaf(r.n * d, d, i & 1 ? r.m2[i / 2].y : r.m2[i / 2].x);
    }
  }
  parts = group_sums(vals, lanes, C, cg, red);
  for (int g = threadIdx.x; g < C / cg; g += kGnThreads) s_m2[g] = sum_parts(red, g, parts);
  __syncthreads();
}

// Sum over the block, for every thread; red: [2][8], used in turn by the parity of `round`.
__device__ __forceinline__ float block_sum(float v, float* red, int round) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  float* to = red + (round & 1) * kGnWarps;
  if (threadIdx.x % 32 == 0) to[threadIdx.x / 32] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int i = 0; i < kGnWarps; ++i) v += to[i];
  return v;
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

__device__ __forceinline__ GnArgs follow(const GnArgs& args) {
  GnArgs a = args;
  const int64_t zero = follow_previous();
  for (const void** p : {&a.x, &a.dout, &a.w, &a.b}) *p = static_cast<const char*>(*p) + zero;
  a.mean += zero, a.rstd += zero, a.part += zero, a.sums += zero;
  return a;
}

using GnRing1 = Ring<8, 1, kGnThreads>;    // forward: 32 KB a block, four blocks per SM
using GnRing2 = Ring<6, 2, kGnThreads>;    // backward (x, dout): 48 KB a block, two blocks per SM

// What a thread does with a position in the forward pass: y = act((x - mu) (rstd w) + b). x - mu comes
// first: folded into the offset, the mean of a map of little variance would cost digits.
template <class T, int ACT>
struct Apply {
  static constexpr int V = Vec<T>::V, P = V / 2;
  float2 A[P], b[P], mu[P];
  __device__ __forceinline__ Apply(const GnArgs& a, int ch, const float* s_mu, const float* s_rs, int g0) {
    load_pairs(static_cast<const T*>(a.w) + ch, A);
    load_pairs(static_cast<const T*>(a.b) + ch, b);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int g1 = (ch + 2 * i) / a.cg - g0, g2 = (ch + 2 * i + 1) / a.cg - g0;
      mu[i] = make_float2(-s_mu[g1], -s_mu[g2]);
      A[i] = mul2(A[i], make_float2(s_rs[g1], s_rs[g2]));
    }
  }
  __device__ __forceinline__ Apply(const GnArgs& a, int ch, float mean, float rstd) {
    load_pairs(static_cast<const T*>(a.w) + ch, A);
    load_pairs(static_cast<const T*>(a.b) + ch, b);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      mu[i] = both(-mean);
      A[i] = mul2(A[i], both(rstd));
    }
  }
  __device__ __forceinline__ void operator()(const uint4& u, T* to) const {
    float2 f[P];
    Vec<T>::unpack(u, f);
#pragma unroll
    for (int i = 0; i < P; ++i) f[i] = act_value<ACT, Vec<T>::exact>(fma2(add2(f[i], mu[i]), A[i], b[i]));
    st_raw(to, Vec<T>::pack(f));
  }
};

template <class T, int ACT>
__global__ void __launch_bounds__(kGnThreads) groupnorm_resident_kernel(const GnArgs args) {
  const GnArgs a = follow(args);
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
  float* red = vals + lanes * a.slab;                                // [max(G, 16)]
  float* s_mean = red + max(G, 2 * kGnWarps);                            // [G], m2 behind it
  const int64_t base = (static_cast<int64_t>(n) * a.HW + p0) * a.C + c0 + col * V;
  const T* x = static_cast<const T*>(a.x) + base;
  const int len = static_cast<int>(p1 - p0);
  Running<V> r;
  if (active) r.walk(x, lane, lanes, len, a.C, [&](int p, const uint4& u) { keep[p * cols + col] = u; });
  T* out = static_cast<T*>(a.out) + base;
  if (G == 1) {
    // one group: block sums of scalars, and every warp joins the cluster's moments by itself
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) m += r.mean[i].x + r.mean[i].y;
    const float here = static_cast<float>(max(len, 1)) * a.cg;
    const float mu_here = block_sum(r.n * m, red, 0) / here;
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float dx = r.mean[i].x - mu_here, dy = r.mean[i].y - mu_here;
      q += fmaf(r.n * dx, dx, r.m2[i].x) + fmaf(r.n * dy, dy, r.m2[i].y);
    }
    const float q_here = block_sum(q, red, 1);
    float mu = mu_here, m2 = q_here;
    if (cl > 1) {
      if (threadIdx.x == 0) s_mean[0] = mu_here, s_mean[1] = q_here;
      cluster_sync_all();
      const int i = static_cast<int>(threadIdx.x) % 32;
      float ni = 0.f, mi = 0.f, qi = 0.f;
      if (i < cl) {
        ni = static_cast<float>(min(a.HW, static_cast<int64_t>(i + 1) * a.span) - min(a.HW, static_cast<int64_t>(i) * a.span)) * a.cg;
        const uint32_t at = mapa_shared(smem_u32(s_mean), i);
        mi = ld_dsmem(at), qi = ld_dsmem(at + 4);
      }
      __syncwarp();
      cluster_arrive();                      // this block has read its peers
      auto warp_sum = [](float v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
      };
      mu = warp_sum(ni * mi) / (static_cast<float>(a.HW) * a.cg);
      m2 = warp_sum(fmaf(ni * (mi - mu), mi - mu, qi));
    }
    const float rs = rsqrtf(m2 / (static_cast<float>(a.HW) * a.cg) + a.eps);
    if (rank == 0 && threadIdx.x == 0 && a.mean != nullptr) {
      const int64_t to = static_cast<int64_t>(n) * (a.C / a.cg) + c0 / a.cg;
      a.mean[to] = mu, a.rstd[to] = rs;
    }
    if (active) {
      const Apply<T, ACT> apply(a, c0 + col * V, mu, rs);
      for (int p = lane; p < len; p += lanes) apply(keep[p * cols + col], out + static_cast<int64_t>(p) * a.C);
    }
    __syncwarp();
    if (cl > 1) cluster_wait();              // no block leaves while its peers may read it
    return;
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
  const Apply<T, ACT> apply(a, c0 + col * V, s_out, s_out + G, c0 / a.cg);
  for (int p = lane; p < len; p += lanes) apply(keep[p * cols + col], out + static_cast<int64_t>(p) * a.C);
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

// The same in the backward pass: xh = (x - mu) rstd, g = dy act'(xh w + b).
template <class T, int ACT>
struct Grad {
  static constexpr int V = Vec<T>::V, P = V / 2;
  float2 w[P], b[P], mu[P], rs[P];
  __device__ __forceinline__ Grad(const GnArgs& a, int n, int ch) {
    load_pairs(static_cast<const T*>(a.w) + ch, w);
    load_pairs(static_cast<const T*>(a.b) + ch, b);
    const int64_t g0 = static_cast<int64_t>(n) * (a.C / a.cg);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int64_t g1 = g0 + (ch + 2 * i) / a.cg, g2 = g0 + (ch + 2 * i + 1) / a.cg;
      rs[i] = make_float2(__ldg(a.rstd + g1), __ldg(a.rstd + g2));
      mu[i] = make_float2(-__ldg(a.mean + g1), -__ldg(a.mean + g2));
    }
  }
  __device__ __forceinline__ void both_terms(int i, const float2& x, const float2& d, float2& xh, float2& g) const {
    xh = mul2(add2(x, mu[i]), rs[i]);
    g = mul2(d, act_slope<ACT, Vec<T>::exact>(fma2(xh, w[i], b[i])));
  }
  __device__ __forceinline__ void sums(const uint4& xu, const uint4& du, float2 (&sg)[P], float2 (&sx)[P]) const {
    float2 f[P], d[P];
    Vec<T>::unpack(xu, f);
    Vec<T>::unpack(du, d);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      float2 xh, g;
      both_terms(i, f[i], d[i], xh, g);
      sg[i] = add2(sg[i], g);
      sx[i] = fma2(g, xh, sx[i]);
    }
  }
  // dx = g (w rstd) + (xh (-rstd m2) + (-rstd m1))
  struct Means {
    float2 k[P], c[P], wr[P];
    __device__ __forceinline__ Means(const Grad& gr, const float* m1, const float* m2, int ch, int cg, int g0) {
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int g1 = (ch + 2 * i) / cg - g0, g2 = (ch + 2 * i + 1) / cg - g0;
        k[i] = mul2(gr.rs[i], make_float2(-m2[g1], -m2[g2]));
        c[i] = mul2(gr.rs[i], make_float2(-m1[g1], -m1[g2]));
        wr[i] = mul2(gr.rs[i], gr.w[i]);
      }
    }
  };
  __device__ __forceinline__ void dx(const Means& m, const uint4& xu, const uint4& du, T* to) const {
    float2 f[P], d[P];
    Vec<T>::unpack(xu, f);
    Vec<T>::unpack(du, d);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      float2 xh, g;
      both_terms(i, f[i], d[i], xh, g);
      f[i] = fma2(g, m.wr[i], fma2(xh, m.k[i], m.c[i]));
    }
    st_raw(to, Vec<T>::pack(f));
  }
};
// a thread's sums into vals [2][lanes][C]
template <int P>
__device__ __forceinline__ void put_sums(float* vals, int lane, int lanes, int C, int ch, const float2 (&sg)[P], const float2 (&sx)[P]) {
#pragma unroll
  for (int i = 0; i < P; ++i) {
    *reinterpret_cast<float2*>(vals + lane * C + ch + 2 * i) = sg[i];
    *reinterpret_cast<float2*>(vals + (lanes + lane) * C + ch + 2 * i) = sx[i];
  }
}

template <class T, int ACT>
__global__ void __launch_bounds__(kGnThreads) groupnorm_bwd_resident_kernel(const GnArgs args) {
  const GnArgs a = follow(args);
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
  const Grad<T, ACT> gr(a, n, c0 + col * V);
  if (active) {
    float2 sg[V / 2], sx[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) sg[i] = sx[i] = both(0.f);
    const T *x = static_cast<const T*>(a.x) + base, *d = static_cast<const T*>(a.dout) + base;
    for (int p = lane; p < len; p += lanes * 2) {
      const bool two = p + lanes < len;
      const int64_t o0 = static_cast<int64_t>(p) * a.C, o1 = static_cast<int64_t>(p + lanes) * a.C;
      uint4 x0 = ld_raw(x + o0), d0 = ld_raw(d + o0), x1, d1;
      if (two) x1 = ld_raw(x + o1), d1 = ld_raw(d + o1);
      keep[p * cols + col] = x0, keep[(a.span + p) * cols + col] = d0;
      gr.sums(x0, d0, sg, sx);
      if (two) {
        keep[(p + lanes) * cols + col] = x1, keep[(a.span + p + lanes) * cols + col] = d1;
        gr.sums(x1, d1, sg, sx);
      }
    }
    put_sums(vals, lane, lanes, S, col * V, sg, sx);
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
  const typename Grad<T, ACT>::Means m(gr, all + 2 * S, all + 2 * S + G, c0 + col * V, a.cg, c0 / a.cg);
  T* dx = static_cast<T*>(a.out) + base;
  for (int p = lane; p < len; p += lanes)
    gr.dx(m, keep[p * cols + col], keep[(a.span + p) * cols + col], dx + static_cast<int64_t>(p) * a.C);
}

// part[n][chunk][g] = mean, squared deviations of the group over the chunk's positions
template <class T>
__global__ void __launch_bounds__(kGnThreads, 4) groupnorm_moments_kernel(const GnArgs args) {
  const GnArgs a = follow(args);
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
    r.walk(x, lane, lanes, static_cast<int>(p1 - p0), a.C, [](int, const uint4&) {});
  }
  block_moments<V>(r, lane < lanes, lane, col, lanes, a.C, a.cg, static_cast<float>(p1 - p0), vals, red, s_mean, s_mean + G);
  for (int g = threadIdx.x; g < G; g += kGnThreads) {
    float* to = a.part + ((static_cast<int64_t>(n) * gridDim.x + blockIdx.x) * G + g) * 2;
    to[0] = s_mean[g], to[1] = s_mean[G + g];
  }
}

// Every block joins its sample's chunks (a warp per group, the same order everywhere) and normalises its own.
template <class T, int ACT>
__global__ void __launch_bounds__(kGnThreads, 4) groupnorm_apply_kernel(const GnArgs args) {
  const GnArgs a = follow(args);
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
  const Apply<T, ACT> apply(a, col * V, gsm, gsm + G, 0);
  const int64_t p0 = static_cast<int64_t>(blockIdx.x) * a.span;
  const int len = static_cast<int>(min(a.HW, p0 + a.span) - p0);
  const int64_t base = (static_cast<int64_t>(n) * a.HW + p0) * a.C + col * V;
  const T* x = static_cast<const T*>(a.x) + base;
  T* out = static_cast<T*>(a.out) + base;
  GnRing1(gsm + (2 * G + 3) / 4 * 4).walk(x, x, lane, lanes, len, a.C, [&](int p, const uint4& u, const uint4&) {
    apply(u, out + static_cast<int64_t>(p) * a.C);
  });
}

// part[n][chunk][0 | 1][c] = sums over the chunk's positions of g and of g xh
template <class T, int ACT>
__global__ void __launch_bounds__(kGnThreads, 2) groupnorm_bwd_sums_kernel(const GnArgs args) {
  const GnArgs a = follow(args);
  constexpr int V = Vec<T>::V;
  extern __shared__ __align__(16) float gsm[];  // [2][lanes][C], [2][C]
  const int cols = a.C / V, lanes = kGnThreads / cols;
  const int col = threadIdx.x % cols, lane = threadIdx.x / cols;
  const int n = a.n0 + blockIdx.y;
  const int64_t p0 = static_cast<int64_t>(blockIdx.x) * a.span;
  if (lane < lanes) {
    const int len = static_cast<int>(min(a.HW, p0 + a.span) - p0);
    const Grad<T, ACT> gr(a, n, col * V);
    float2 sg[V / 2], sx[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) sg[i] = sx[i] = both(0.f);
    const int64_t base = (static_cast<int64_t>(n) * a.HW + p0) * a.C + col * V;
    const T *x = static_cast<const T*>(a.x) + base, *d = static_cast<const T*>(a.dout) + base;
    GnRing2(gsm + (2 * lanes + 2) * a.C).walk(x, d, lane, lanes, len, a.C, [&](int, const uint4& xu, const uint4& du) {
      gr.sums(xu, du, sg, sx);
    });
    put_sums(gsm, lane, lanes, a.C, col * V, sg, sx);
  }
  float* tot = gsm + 2 * lanes * a.C;
  channel_totals(gsm, lanes, a.C, tot);
  float* to = a.part + (static_cast<int64_t>(n) * gridDim.x + blockIdx.x) * 2 * a.C;
  for (int e = threadIdx.x; e < 2 * a.C; e += kGnThreads) to[e] = tot[e];
}

// sums[n][..] = the sample's chunks; a warp's lanes are 32 entries, its block's warps share the chunks
__global__ void __launch_bounds__(1024) groupnorm_bwd_totals_kernel(const float* part, int n0, int chunks, int C, float* sums) {
  part += follow_previous();
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
__global__ void __launch_bounds__(kGnThreads, 2) groupnorm_bwd_dx_kernel(const GnArgs args) {
  const GnArgs a = follow(args);
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
  const Grad<T, ACT> gr(a, n, col * V);
  const typename Grad<T, ACT>::Means m(gr, gsm + 2 * a.C, gsm + 2 * a.C + G, col * V, a.cg, 0);
  const int64_t p0 = static_cast<int64_t>(blockIdx.x) * a.span;
  const int len = static_cast<int>(min(a.HW, p0 + a.span) - p0);
  const int64_t base = (static_cast<int64_t>(n) * a.HW + p0) * a.C + col * V;
  const T *x = static_cast<const T*>(a.x) + base, *d = static_cast<const T*>(a.dout) + base;
  T* dx = static_cast<T*>(a.out) + base;
  GnRing2(gsm + (2 * (a.C + G) + 3) / 4 * 4).walk(x, d, lane, lanes, len, a.C, [&](int p, const uint4& xu, const uint4& du) {
    gr.dx(m, xu, du, dx + static_cast<int64_t>(p) * a.C);
  });
}

// db[c] = sum over the P partials of sums[p][0][c], dw[c] of sums[p][1][c]
template <class T>
__global__ void __launch_bounds__(1024) norm_param_grad_kernel(const float* __restrict__ sums, int P, int C,
                                                               T* __restrict__ dw, T* __restrict__ db) {
  sums += follow_previous();
  __shared__ float sm[32][33];
  const int e = blockIdx.x * 32 + threadIdx.x;
  float s = 0.f;
  if (e < 2 * C) {
#pragma unroll 8
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
                  : keep + (static_cast<size_t>(lanes) * slab + std::max(G, 2 * kGnWarps) + 2 * G) * 4;
}

static GnPlan groupnorm_plan(int N, int64_t HW, int C, int groups, int elem, bool backward, int most = 8) {
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
  const int64_t span0 = (HW + cl - 1) / cl;
  // 16 blocks (not portable) only shorten the walk: they change neither what fits nor the workspace
  if (most >= 16 && cl == 8 && clusters * 16 <= 148 && HW > 16 * 64) cl = 16;
  const int64_t span = (HW + cl - 1) / cl;
  if (room && span0 < (1 << 20) && gn_resident_smem(span0, slab, cg, elem, backward) <= static_cast<size_t>(kGnResident)) {
    p.slab = slab, p.cluster = cl, p.span = static_cast<int>(span);
    p.smem = gn_resident_smem(span, slab, cg, elem, backward);
    return p;
  }
  const int64_t sample = HW * C * elem * (backward ? 2 : 1);
  const int64_t fit = std::max<int64_t>(1, std::min<int64_t>(N, kGnL2 / sample)), launches = (N + fit - 1) / fit;
  p.batch = static_cast<int>((N + launches - 1) / launches);             // launches of about equal size
  const int per_sm = backward ? 2 : 4;
  const int64_t want = std::max<int64_t>(1, 148 * per_sm / p.batch);   // one wave: a block more would be a second
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
  if (C % V || C / V > kGnThreads || N > 65535 || HW >= (1ll << 31)) return SSAM_ERR_UNSUPPORTED;
  const size_t need = groupnorm_workspace_size(N, HW, C, G, dtype, backward);
  if (workspace_bytes < need || (need > 0 && workspace == nullptr)) return SSAM_ERR_INVALID;
  return SSAM_OK;
}

template <class K>
static int launch_gn(K kernel, PerDeviceOnce& once, dim3 grid, size_t smem, int cluster, cudaStream_t stream,
                     const GnArgs& a) {
  const int st = allow_smem(once, kernel, kGnResident);
  if (st != SSAM_OK) return st;
  return launch_following(kernel, grid, dim3(kGnThreads), smem, cluster, stream, a);
}
static size_t gn_floats(size_t n) { return (n + 3) / 4 * 16; }

template <class T, int ACT>
static int groupnorm_fwd_t(GnArgs a, int N, int G, float* ws, cudaStream_t stream) {
  static PerDeviceOnce resident, moments, apply;
  static ClusterLimit limit;
  const GnPlan p = groupnorm_plan(N, a.HW, a.C, G, sizeof(T), false,
                                  limit.get(groupnorm_resident_kernel<T, ACT>, kGnThreads, kGnResident));
  a.span = p.span, a.slab = p.slab, a.part = ws;
  if (p.cluster)
    return launch_gn(groupnorm_resident_kernel<T, ACT>, resident, dim3(p.cluster, a.C / p.slab, N), p.smem, p.cluster,
                     stream, a);
  const int lanes = kGnThreads / (a.C / Vec<T>::V);
  for (a.n0 = 0; a.n0 < N; a.n0 += p.batch) {
    const dim3 grid(p.chunks, std::min(p.batch, N - a.n0));
    int st = launch_gn(groupnorm_moments_kernel<T>, moments, grid,
                       gn_floats(lanes * a.C + std::max(G, kGnWarps) + 2 * G), 1, stream, a);
    if (st == SSAM_OK)
      st = launch_gn(groupnorm_apply_kernel<T, ACT>, apply, grid, gn_floats(2 * G) + GnRing1::bytes, 1, stream, a);
    if (st != SSAM_OK) return st;
  }
  return SSAM_OK;
}

template <class T, int ACT>
static int groupnorm_bwd_t(GnArgs a, int N, int G, void* dw, void* db, float* ws, cudaStream_t stream) {
  static PerDeviceOnce resident, sums, dx;
  static ClusterLimit limit;
  const GnPlan p = groupnorm_plan(N, a.HW, a.C, G, sizeof(T), true,
                                  limit.get(groupnorm_bwd_resident_kernel<T, ACT>, kGnThreads, kGnResident));
  a.span = p.span, a.slab = p.slab, a.sums = ws;
  a.part = ws + gn_align(static_cast<size_t>(N) * 2 * a.C * sizeof(float)) / sizeof(float);
  int st;
  if (p.cluster) {
    st = launch_gn(groupnorm_bwd_resident_kernel<T, ACT>, resident, dim3(p.cluster, a.C / p.slab, N), p.smem, p.cluster,
                   stream, a);
    if (st != SSAM_OK) return st;
  } else {
    const int lanes = kGnThreads / (a.C / Vec<T>::V);
    for (a.n0 = 0; a.n0 < N; a.n0 += p.batch) {
      const dim3 grid(p.chunks, std::min(p.batch, N - a.n0));
      st = launch_gn(groupnorm_bwd_sums_kernel<T, ACT>, sums, grid, gn_floats((2 * lanes + 2) * a.C) + GnRing2::bytes, 1,
                     stream, a);
      if (st != SSAM_OK) return st;
      st = launch_following(groupnorm_bwd_totals_kernel, dim3((2 * a.C + 31) / 32, grid.y), dim3(32, 32), 0, 1, stream, a.part, a.n0,
                            p.chunks, a.C, a.sums);
      if (st == SSAM_OK)
        st = launch_gn(groupnorm_bwd_dx_kernel<T, ACT>, dx, grid, gn_floats(2 * (a.C + G)) + GnRing2::bytes, 1, stream, a);
      if (st != SSAM_OK) return st;
    }
  }
  return launch_following(norm_param_grad_kernel<T>, dim3((2 * a.C + 31) / 32), dim3(32, 32), 0, 1, stream, a.sums, N, a.C,
                          static_cast<T*>(dw), static_cast<T*>(db));
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
// rows' parameter gradients into one partial. 262144 x 64 with GELU, fp16: 51 us with the forward pass
// (2.6 TB/s), issuing in 58 % of the cycles at 30 % of the warps; 4096 x 256 without it 8.1 us, three launches.
// ---------------------------------------------------------------------------
constexpr int kLnRing = 3;
using LnRing = Ring<kLnRing, 2, 256>;      // 24 KB a block

template <class T, int C, bool GELU>
__global__ void __launch_bounds__(256) layernorm_half_bwd_kernel(const T* __restrict__ x, const T* __restrict__ dout,
                                                                 int64_t rows, const T* __restrict__ w,
                                                                 const T* __restrict__ b, float eps, T* __restrict__ dx,
                                                                 float* __restrict__ sums) {
  const int64_t zero = follow_previous();
  x += zero, dout += zero, w += zero, b += zero;
  constexpr int TPR = C / 8, RPB = 256 / TPR;
  __shared__ __align__(16) float part[2][RPB][C];
  const int t = threadIdx.x % TPR, lr = threadIdx.x / TPR;
  float2 wf[4], bf[4], sg[4], sx[4];
  load_pairs(w + t * 8, wf);
  load_pairs(b + t * 8, bf);
#pragma unroll
  for (int i = 0; i < 4; ++i) sg[i] = sx[i] = both(0.f);
  auto row_sum = [](float2 p) {
    float v = p.x + p.y;
#pragma unroll
    for (int o = 1; o < TPR; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v * (1.f / C);
  };
  __shared__ __align__(16) uint4 ring_mem[LnRing::bytes / 16];
  const LnRing ring(ring_mem);
  const int64_t step = static_cast<int64_t>(gridDim.x) * RPB;
  auto request = [&](int slot, int64_t row) {
    if (row < rows) {
      ring.fetch(slot, 0, x + row * C + t * 8);
      ring.fetch(slot, 1, dout + row * C + t * 8);
    }
    LnRing::commit();
  };
  int64_t r = static_cast<int64_t>(blockIdx.x) * RPB + lr;
#pragma unroll
  for (int i = 0; i < kLnRing; ++i) request(i, r + i * step);
  int slot = 0;
  // a warp's lanes hold whole rows: all of a row's lanes are behind the end together, and the others go on
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * RPB; r0 < rows; r0 += step, r += step) {
    float2 f[4], d[4], s = both(0.f);
    LnRing::wait();
    const uint4 none = make_uint4(0u, 0u, 0u, 0u);
    Vec<T>::unpack(r < rows ? ring.get(slot, 0) : none, f);
    Vec<T>::unpack(r < rows ? ring.get(slot, 1) : none, d);
#pragma unroll
    for (int i = 0; i < 4; ++i) s = add2(s, f[i]);
    const float mu = row_sum(s);
    s = both(0.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = add2(f[i], both(-mu)), s = fma2(f[i], f[i], s);
    const float rs = rsqrtf(row_sum(s) + eps);
    float2 s1 = both(0.f), s2 = both(0.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = mul2(f[i], both(rs));
      if (GELU) d[i] = mul2(d[i], gelu_slope2(fma2(f[i], wf[i], bf[i])));
      sg[i] = add2(sg[i], d[i]);
      sx[i] = fma2(d[i], f[i], sx[i]);
      d[i] = mul2(d[i], wf[i]);
      s1 = add2(s1, d[i]);
      s2 = fma2(d[i], f[i], s2);
    }
    const float m1 = -rs * row_sum(s1), m2 = -rs * row_sum(s2);
    if (r < rows) {
#pragma unroll
      for (int i = 0; i < 4; ++i) d[i] = fma2(d[i], both(rs), fma2(f[i], both(m2), both(m1)));
      st_raw(dx + r * C + t * 8, Vec<T>::pack(d));
    }
    request(slot, r + kLnRing * step);
    slot = slot + 1 == kLnRing ? 0 : slot + 1;
  }
  put_sums(&part[0][0][0], lr, RPB, C, t * 8, sg, sx);
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * C; c += 256) {
    float s = 0.f;
#pragma unroll 8
    for (int k = 0; k < RPB; ++k) s += part[c / C][k][c % C];
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
  const int st = launch_following(kernel, dim3(blocks), dim3(256), 0, 1, stream, static_cast<const T*>(x),
                                  static_cast<const T*>(dout), rows, static_cast<const T*>(w), static_cast<const T*>(b), eps,
                                  static_cast<T*>(dx), ws);
  if (st != SSAM_OK) return st;
  return launch_following(norm_param_grad_kernel<T>, dim3((2 * C + 31) / 32), dim3(32, 32), 0, 1, stream, ws, blocks, C,
                          static_cast<T*>(dw), static_cast<T*>(db));
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
