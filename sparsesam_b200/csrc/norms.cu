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

// act(z), and act'(z) through *slope. GELU is the erf form.
template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  if (ACT == kActRelu) return z < 0.f ? 0.f : z;  // NaN stays NaN
  if (ACT == kActGelu) return 0.5f * z * (1.f + erff(z * 0.70710678118654752440f));
  if (ACT == kActSilu) return z / (1.f + expf(-z));
  return z;
}
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if (ACT == kActRelu) return z > 0.f ? 1.f : 0.f;
  if (ACT == kActGelu)
    return 0.5f * (1.f + erff(z * 0.70710678118654752440f)) + z * expf(-0.5f * z * z) * 0.39894228040143267794f;
  if (ACT == kActSilu) {
    const float s = 1.f / (1.f + expf(-z));
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
  static __device__ __forceinline__ void load(const float* p, float (&f)[4]) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
  }
  static __device__ __forceinline__ void store(float* p, const float (&f)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  }
  static __device__ __forceinline__ float round(float f) { return f; }
};
template <>
struct Vec<__half> {
  static constexpr int V = 8;
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

// (count, mean, sum of squared deviations) of a set of values
struct Moments {
  float n, mean, m2;
};
__device__ __forceinline__ Moments merge(Moments a, Moments b) {
  const float n = a.n + b.n;
  if (n == 0.f) return a;
  const float f = b.n / n, d = b.mean - a.mean;
  return {n, fmaf(d, f, a.mean), a.m2 + b.m2 + d * d * a.n * f};
}

// ---------------------------------------------------------------------------
// GroupNorm. A block handles `span` positions of one sample; its threads form
// `lanes` = 256 / cols position lanes of cols = C / V vector columns.
// ---------------------------------------------------------------------------
constexpr int kGnThreads = 256;
constexpr int kGnBatch = 4;  // positions whose moments are computed exactly, then merged

// moments[n][chunk][g] of each group over the chunk's positions
template <class T>
__global__ void __launch_bounds__(kGnThreads) groupnorm_stats_kernel(const T* __restrict__ x, int64_t HW, int C, int G,
                                                                     int span, float* __restrict__ moments) {
  constexpr int V = Vec<T>::V;
  extern __shared__ float gsm[];  // [lanes][C] x (mean, m2), then [lanes] counts
  const int cols = C / V, lanes = kGnThreads / cols;
  const int col = threadIdx.x % cols, lane = threadIdx.x / cols;
  const int n = blockIdx.y, chunk = blockIdx.x;
  const int64_t p0 = static_cast<int64_t>(chunk) * span, p1 = min(HW, p0 + span);
  float *s_mean = gsm, *s_m2 = gsm + lanes * C, *s_n = s_m2 + lanes * C;
  if (lane < lanes) {
    float mean[V], m2[V], cnt = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) mean[i] = 0.f, m2[i] = 0.f;
    const T* base = x + static_cast<int64_t>(n) * HW * C + col * V;
    for (int64_t p = p0 + lane; p < p1; p += lanes * kGnBatch) {
      float f[kGnBatch][V];
      int k = 0;
#pragma unroll
      for (int j = 0; j < kGnBatch; ++j) {
        if (p + static_cast<int64_t>(j) * lanes < p1) {
          Vec<T>::load(base + (p + static_cast<int64_t>(j) * lanes) * C, f[j]);
          k = j + 1;
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) f[j][i] = 0.f;
        }
      }
      const float inv = 1.f / k, nn = cnt + k, w = k / nn, cw = cnt * w;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float s = 0.f, q = 0.f;
#pragma unroll
        for (int j = 0; j < kGnBatch; ++j) s += f[j][i];
        s *= inv;
#pragma unroll
        for (int j = 0; j < kGnBatch; ++j) {
          const float d = j < k ? f[j][i] - s : 0.f;
          q = fmaf(d, d, q);
        }
        const float d = s - mean[i];
        mean[i] = fmaf(d, w, mean[i]);
        m2[i] += fmaf(d * d, cw, q);
      }
      cnt = nn;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) s_mean[lane * C + col * V + i] = mean[i], s_m2[lane * C + col * V + i] = m2[i];
    if (col == 0) s_n[lane] = cnt;
  }
  __syncthreads();
  // per channel over the lanes, in place in lane 0's slots
  for (int c = threadIdx.x; c < C; c += kGnThreads) {
    Moments a = {s_n[0], s_mean[c], s_m2[c]};
    for (int l = 1; l < lanes; ++l) a = merge(a, {s_n[l], s_mean[l * C + c], s_m2[l * C + c]});
    s_mean[c] = a.mean, s_m2[c] = a.m2;
  }
  __syncthreads();
  const int cg = C / G;
  const float per = static_cast<float>(p1 - p0);
  for (int g = threadIdx.x; g < G; g += kGnThreads) {
    Moments a = {per, s_mean[g * cg], s_m2[g * cg]};
    for (int c = 1; c < cg; ++c) a = merge(a, {per, s_mean[g * cg + c], s_m2[g * cg + c]});
    float* to = moments + ((static_cast<int64_t>(n) * gridDim.x + chunk) * G + g) * 2;
    to[0] = a.mean, to[1] = a.m2;
  }
}

// Each block merges its sample's chunk moments (the same order everywhere) and normalises its chunk.
template <class T, int ACT>
__global__ void __launch_bounds__(kGnThreads)
    groupnorm_apply_kernel(const T* __restrict__ x, int64_t HW, int C, int G, int span, const float* __restrict__ moments,
                           const T* __restrict__ w, const T* __restrict__ b, float eps, T* __restrict__ out,
                           float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  constexpr int V = Vec<T>::V;
  extern __shared__ float gsm[];  // [G] mean, [G] rstd
  const int n = blockIdx.y, chunks = gridDim.x, cg = C / G;
  for (int g = threadIdx.x; g < G; g += kGnThreads) {
    Moments a = {0.f, 0.f, 0.f};
    for (int k = 0; k < chunks; ++k) {
      const float* m = moments + ((static_cast<int64_t>(n) * chunks + k) * G + g) * 2;
      const int64_t len = min(HW - static_cast<int64_t>(k) * span, static_cast<int64_t>(span));
      a = merge(a, {static_cast<float>(len) * cg, m[0], m[1]});
    }
    const float rstd = rsqrtf(a.m2 / a.n + eps);
    gsm[g] = a.mean, gsm[G + g] = rstd;
    if (blockIdx.x == 0 && mean_out != nullptr) {
      mean_out[static_cast<int64_t>(n) * G + g] = a.mean;
      rstd_out[static_cast<int64_t>(n) * G + g] = rstd;
    }
  }
  __syncthreads();
  const int cols = C / V, lanes = kGnThreads / cols;
  const int col = threadIdx.x % cols, lane = threadIdx.x / cols;
  if (lane >= lanes) return;
  float mu[V], rs[V], wf[V], bf[V];
  Vec<T>::load(w + col * V, wf);
  Vec<T>::load(b + col * V, bf);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int g = (col * V + i) / cg;
    mu[i] = gsm[g], rs[i] = gsm[G + g];
  }
  const int64_t p0 = static_cast<int64_t>(blockIdx.x) * span, p1 = min(HW, p0 + span);
  const int64_t base = static_cast<int64_t>(n) * HW * C + col * V;
  for (int64_t p = p0 + lane; p < p1; p += lanes) {
    float f[V];
    Vec<T>::load(x + base + p * C, f);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = act_value<ACT>(fmaf((f[i] - mu[i]) * rs[i], wf[i], bf[i]));
    Vec<T>::store(out + base + p * C, f);
  }
}

// sums[n][chunk][0 | 1][c] = sum over the chunk's positions of g and of g xh
template <class T, int ACT>
__global__ void __launch_bounds__(kGnThreads)
    groupnorm_bwd_sums_kernel(const T* __restrict__ x, const T* __restrict__ dout, int64_t HW, int C, int G, int span,
                              const T* __restrict__ w, const T* __restrict__ b, const float* __restrict__ mean,
                              const float* __restrict__ rstd, float* __restrict__ sums) {
  constexpr int V = Vec<T>::V;
  extern __shared__ float gsm[];  // [lanes][2][C]
  const int cols = C / V, lanes = kGnThreads / cols, cg = C / G;
  const int col = threadIdx.x % cols, lane = threadIdx.x / cols;
  const int n = blockIdx.y;
  const int64_t p0 = static_cast<int64_t>(blockIdx.x) * span, p1 = min(HW, p0 + span);
  if (lane < lanes) {
    float mu[V], rs[V], wf[V], bf[V], sg[V], sx[V];
    Vec<T>::load(w + col * V, wf);
    Vec<T>::load(b + col * V, bf);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int64_t g = static_cast<int64_t>(n) * G + (col * V + i) / cg;
      mu[i] = mean[g], rs[i] = rstd[g], sg[i] = 0.f, sx[i] = 0.f;
    }
    const int64_t base = static_cast<int64_t>(n) * HW * C + col * V;
    for (int64_t p = p0 + lane; p < p1; p += lanes) {
      float f[V], d[V];
      Vec<T>::load(x + base + p * C, f);
      Vec<T>::load(dout + base + p * C, d);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float xh = (f[i] - mu[i]) * rs[i];
        const float g = d[i] * act_slope<ACT>(fmaf(xh, wf[i], bf[i]));
        sg[i] += g;
        sx[i] = fmaf(g, xh, sx[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      gsm[(lane * 2) * C + col * V + i] = sg[i];
      gsm[(lane * 2 + 1) * C + col * V + i] = sx[i];
    }
  }
  __syncthreads();
  float* to = sums + (static_cast<int64_t>(n) * gridDim.x + blockIdx.x) * 2 * C;
  for (int c = threadIdx.x; c < 2 * C; c += kGnThreads) {
    float s = 0.f;
    for (int l = 0; l < lanes; ++l) s += gsm[l * 2 * C + c];
    to[c] = s;
  }
}

template <class T, int ACT>
__global__ void __launch_bounds__(kGnThreads)
    groupnorm_bwd_dx_kernel(const T* __restrict__ x, const T* __restrict__ dout, int64_t HW, int C, int G, int span,
                            const T* __restrict__ w, const T* __restrict__ b, const float* __restrict__ mean,
                            const float* __restrict__ rstd, const float* __restrict__ sums, T* __restrict__ dx) {
  constexpr int V = Vec<T>::V;
  extern __shared__ float gsm[];  // [2][C] channel sums times w, [2][G] group means
  const int n = blockIdx.y, chunks = gridDim.x, cg = C / G;
  for (int c = threadIdx.x; c < 2 * C; c += kGnThreads) {
    float s = 0.f;
    for (int k = 0; k < chunks; ++k) s += sums[(static_cast<int64_t>(n) * chunks + k) * 2 * C + c];
    gsm[c] = s * static_cast<float>(w[c % C]);
  }
  __syncthreads();
  for (int g = threadIdx.x; g < 2 * G; g += kGnThreads) {
    float s = 0.f;
    for (int c = 0; c < cg; ++c) s += gsm[g / G * C + g % G * cg + c];
    gsm[2 * C + g] = s / (static_cast<float>(HW) * cg);
  }
  __syncthreads();
  const int cols = C / V, lanes = kGnThreads / cols;
  const int col = threadIdx.x % cols, lane = threadIdx.x / cols;
  if (lane >= lanes) return;
  float mu[V], rs[V], wf[V], bf[V], m1[V], m2[V];
  Vec<T>::load(w + col * V, wf);
  Vec<T>::load(b + col * V, bf);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int g = (col * V + i) / cg;
    mu[i] = mean[static_cast<int64_t>(n) * G + g], rs[i] = rstd[static_cast<int64_t>(n) * G + g];
    m1[i] = gsm[2 * C + g], m2[i] = gsm[2 * C + G + g];
  }
  const int64_t p0 = static_cast<int64_t>(blockIdx.x) * span, p1 = min(HW, p0 + span);
  const int64_t base = static_cast<int64_t>(n) * HW * C + col * V;
  for (int64_t p = p0 + lane; p < p1; p += lanes) {
    float f[V], d[V];
    Vec<T>::load(x + base + p * C, f);
    Vec<T>::load(dout + base + p * C, d);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float xh = (f[i] - mu[i]) * rs[i];
      const float gw = d[i] * act_slope<ACT>(fmaf(xh, wf[i], bf[i])) * wf[i];
      f[i] = rs[i] * (gw - m1[i] - xh * m2[i]);
    }
    Vec<T>::store(dx + base + p * C, f);
  }
}

// db[c] = sum over the P partials of sums[p][0][c], dw[c] of sums[p][1][c]; one warp per 1 entry column.
template <class T>
__global__ void norm_param_grad_kernel(const float* __restrict__ sums, int64_t P, int C, T* __restrict__ dw,
                                       T* __restrict__ db) {
  __shared__ float part[8][33];
  const int c = blockIdx.x * 32 + threadIdx.x;  // 0 .. 2C
  float s = 0.f;
  if (c < 2 * C)
    for (int64_t p = threadIdx.y; p < P; p += 8) s += sums[p * 2 * C + c];
  part[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < 2 * C) {
    for (int k = 1; k < 8; ++k) s += part[k][threadIdx.x];
    norm_store1(c < C ? db + c : dw + (c - C), s);
  }
}

static size_t gn_align(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }

// Positions per block: about two waves of blocks over the device, at least 32 positions each.
static int groupnorm_span(int N, int64_t HW) {
  const int64_t want = std::max<int64_t>(1, 4 * 148 / N);
  const int64_t span = std::max<int64_t>(32, (HW + want - 1) / want);
  return static_cast<int>(std::min<int64_t>(span, 1 << 24));
}
static int64_t groupnorm_chunks(int N, int64_t HW) {
  const int span = groupnorm_span(N, HW);
  return (HW + span - 1) / span;
}

size_t groupnorm_workspace_size(int N, int64_t HW, int C, int groups, int backward) {
  if (N <= 0 || HW <= 0 || C <= 0 || groups <= 0) return 0;
  const size_t per = backward ? 2 * static_cast<size_t>(C) : 2 * static_cast<size_t>(groups);
  return gn_align(static_cast<size_t>(N) * groupnorm_chunks(N, HW) * per * sizeof(float));
}

static int groupnorm_check(int N, int64_t HW, int C, int G, int act, int dtype, size_t workspace_bytes,
                           const void* workspace, int backward) {
  if (N <= 0 || HW <= 0 || C <= 0 || G <= 0 || C % G || act < 0 || act > 3 || dtype < 0 || dtype > 2)
    return SSAM_ERR_INVALID;
  const int V = dtype == 2 ? 4 : 8;
  if (C % V || C / V > kGnThreads || N > 65535 || HW > (1ll << 31)) return SSAM_ERR_UNSUPPORTED;
  if (workspace == nullptr || workspace_bytes < groupnorm_workspace_size(N, HW, C, G, backward)) return SSAM_ERR_INVALID;
  return SSAM_OK;
}

template <class T, int ACT>
static int groupnorm_fwd_t(const void* x, int N, int64_t HW, int C, int G, const void* w, const void* b, float eps,
                           void* out, float* mean, float* rstd, float* ws, cudaStream_t stream) {
  const int span = groupnorm_span(N, HW);
  const dim3 grid(static_cast<unsigned>(groupnorm_chunks(N, HW)), N);
  const int lanes = kGnThreads / (C / Vec<T>::V);
  const size_t smem = (2 * static_cast<size_t>(lanes) * C + lanes) * sizeof(float);
  groupnorm_stats_kernel<T><<<grid, kGnThreads, smem, stream>>>(static_cast<const T*>(x), HW, C, G, span, ws);
  int st = status_from_cuda(cudaGetLastError());
  if (st != SSAM_OK) return st;
  groupnorm_apply_kernel<T, ACT><<<grid, kGnThreads, 2 * G * sizeof(float), stream>>>(
      static_cast<const T*>(x), HW, C, G, span, ws, static_cast<const T*>(w), static_cast<const T*>(b), eps,
      static_cast<T*>(out), mean, rstd);
  return status_from_cuda(cudaGetLastError());
}

template <class T, int ACT>
static int groupnorm_bwd_t(const void* x, const void* dout, int N, int64_t HW, int C, int G, const void* w,
                           const void* b, const float* mean, const float* rstd, void* dx, void* dw, void* db, float* ws,
                           cudaStream_t stream) {
  const int span = groupnorm_span(N, HW);
  const dim3 grid(static_cast<unsigned>(groupnorm_chunks(N, HW)), N);
  const int lanes = kGnThreads / (C / Vec<T>::V);
  const T *xt = static_cast<const T*>(x), *dt = static_cast<const T*>(dout), *wt = static_cast<const T*>(w),
          *bt = static_cast<const T*>(b);
  groupnorm_bwd_sums_kernel<T, ACT><<<grid, kGnThreads, 2 * static_cast<size_t>(lanes) * C * sizeof(float), stream>>>(
      xt, dt, HW, C, G, span, wt, bt, mean, rstd, ws);
  int st = status_from_cuda(cudaGetLastError());
  if (st != SSAM_OK) return st;
  groupnorm_bwd_dx_kernel<T, ACT><<<grid, kGnThreads, 2 * static_cast<size_t>(C + G) * sizeof(float), stream>>>(
      xt, dt, HW, C, G, span, wt, bt, mean, rstd, ws, static_cast<T*>(dx));
  st = status_from_cuda(cudaGetLastError());
  if (st != SSAM_OK) return st;
  norm_param_grad_kernel<T><<<(2 * C + 31) / 32, dim3(32, 8), 0, stream>>>(
      ws, static_cast<int64_t>(N) * grid.x, C, static_cast<T*>(dw), static_cast<T*>(db));
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
  float* ws = static_cast<float*>(workspace);
#define ARGS (x, N, HW, C, groups, w, b, eps, out, mean, rstd, ws, stream)
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
  float* ws = static_cast<float*>(workspace);
#define ARGS (x, dout, N, HW, C, groups, w, b, mean, rstd, dx, dw, db, ws, stream)
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
      const float g = GELU ? d[i] * act_slope<kActGelu>(fmaf(f[i], wf[i], bf[i])) : d[i];
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
  norm_param_grad_kernel<T><<<(2 * C + 31) / 32, dim3(32, 8), 0, stream>>>(ws, blocks, C, static_cast<T*>(dw),
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
