// Cross attention between two token sets of different lengths (prompt tokens <->
// image tokens in the mask decoder), forward and backward.
//
//   S[r, j] = scale <q_r, k_j>,  P = softmax over the keys that are there,  O = P V
//   dV = P^T dO,  dP = dO V^T,  D_r = sum_j P dP = <dO_r, O_r>,
//   dS = P (dP - D),  dQ = scale dS K,  dK = scale dS^T Q
//
// q (B, Tq, heads, d), k and v (B, Tk, kv_heads, d): kv_heads divides heads, and
// query head h reads key head h / (heads / kv_heads). The query heads of one key
// head are handled as further query rows: row r = g Tq + t of key head n is token t
// of head n * group + g. Keys at or behind key_lens[b], and keys whose key_mask
// byte is 0, are not there: their logits are never used and their K and V rows are
// read as zeros, so whatever they hold (infinities, NaN) reaches no result. A query
// without keys gives a zero row and zero gradients.
//
// Softmax statistics are kept in base 2: m = max of scale log2(e) s, and
// lse = m + log2(sum 2^(.. - m)), +infinity for a row without keys, which makes
// every probability of that row 2^-inf = 0 in the backward pass.
//
// Work along the long axis is split over the slices of a block and over the blocks
// of a cluster; the partial results meet in (distributed) shared memory in a fixed
// order, so results do not depend on scheduling and no workspace is needed.
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "host_util.h"

namespace ssam {

struct XAttn {
  const void *q, *k, *v, *dout;
  int64_t qs[3], ks[3], vs[3], os[3];  // element strides (batch, token, head); os: out / dout
  int B, Tq, Tk, heads, kv_heads, group, d;
  float scale, c;                      // c = scale * log2(e)
  const int32_t* key_lens;
  const uint8_t* key_mask;             // [B, Tk]
  void* out;
  float* out_f32;                      // [B, Tq, heads, d]
  float* lse;                          // [B, heads, Tq]
  float* delta;                        // [B, heads, Tq]
  void *dq, *dk, *dv;                  // contiguous
};

__device__ __forceinline__ int xattn_keys(const XAttn& a, int b) {
  return a.key_lens == nullptr ? a.Tk : min(max(__ldg(a.key_lens + b), 0), a.Tk);
}

// cluster-wide helpers
__device__ __forceinline__ uint32_t cluster_nctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ float ld_dsmem(uint32_t cluster_addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
  return v;
}

__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <class K>
static int launch_cluster(K kernel, dim3 grid, int threads, size_t smem, int cluster, cudaStream_t stream,
                          const XAttn& a, int arg) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return status_from_cuda(cudaLaunchKernelEx(&cfg, kernel, a, arg));
}

}  // namespace ssam

#include "cross_attention_mma.cuh"

namespace ssam {

// ---------------------------------------------------------------------------
// fp32 inputs: scalar kernels (fp32 FMAs). A thread owns DT dims of one row, TPR threads share
// a row. A block holds RB rows x KS slices of the other axis (RB * KS * TPR = 128).
// ---------------------------------------------------------------------------
constexpr int kXThreads = 128;
constexpr int kXTile = 32;  // entries of the other axis staged at a time

template <int DT, int TPR>
__device__ __forceinline__ float row_dot(const float (&a)[DT], const float* b) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < DT; i += 4) {
    const float4 v = *reinterpret_cast<const float4*>(b + i);
    s = fmaf(a[i], v.x, s);
    s = fmaf(a[i + 1], v.y, s);
    s = fmaf(a[i + 2], v.z, s);
    s = fmaf(a[i + 3], v.w, s);
  }
#pragma unroll
  for (int o = 1; o < TPR; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}
template <int DT>
__device__ __forceinline__ void row_axpy(float w, const float* b, float (&acc)[DT]) {
#pragma unroll
  for (int i = 0; i < DT; i += 4) {
    const float4 v = *reinterpret_cast<const float4*>(b + i);
    acc[i] = fmaf(w, v.x, acc[i]);
    acc[i + 1] = fmaf(w, v.y, acc[i + 1]);
    acc[i + 2] = fmaf(w, v.z, acc[i + 2]);
    acc[i + 3] = fmaf(w, v.w, acc[i + 3]);
  }
}
template <int DT>
__device__ __forceinline__ void load_row(const float* p, int dims, bool ok, float (&r)[DT]) {
#pragma unroll
  for (int i = 0; i < DT; i += 4) {
    const float4 v = ok && i < dims ? __ldg(reinterpret_cast<const float4*>(p + i)) : make_float4(0.f, 0.f, 0.f, 0.f);
    r[i] = v.x, r[i + 1] = v.y, r[i + 2] = v.z, r[i + 3] = v.w;
  }
}

// Copies `n` rows (<= kXTile) of width d into sm[kXTile][LD] as floats; rows for
// which ok(i) is false, and channels past d, are zero.
template <int DP, class P, class O>
__device__ __forceinline__ void stage_rows(float* sm, int n, int d, P row, O ok) {
  constexpr int V = DP / 4, LD = DP + 4;
  for (int e = threadIdx.x; e < kXTile * V; e += kXThreads) {
    const int i = e / V, c = (e % V) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < n && c < d && ok(i)) v = __ldg(reinterpret_cast<const float4*>(row(i) + c));
    *reinterpret_cast<float4*>(sm + i * LD + c) = v;
  }
}

// Sum over the KS slices of the block and the blocks of the cluster of part[slice][row][W]:
// the block's slices are summed into slice 0, then the cluster's blocks each take a share
// of the (row, column) entries. emit(row, col, sum) is called once per entry.
template <class E>
__device__ __forceinline__ void merge_sums(float* part, int KS, int RB, int W, E emit) {
  __syncthreads();
  const int n = RB * W;
  for (int e = threadIdx.x; e < n; e += kXThreads) {
    float s = part[e];
    for (int i = 1; i < KS; ++i) s += part[i * n + e];
    part[e] = s;
  }
  const uint32_t cl = cluster_nctarank(), rank = cluster_ctarank();
  if (cl == 1) {
    __syncthreads();
    for (int e = threadIdx.x; e < n; e += kXThreads) emit(e / W, e % W, part[e]);
    return;
  }
  cluster_sync_all();
  const uint32_t base = smem_u32(part);
  for (int e = rank * kXThreads + threadIdx.x; e < n; e += cl * kXThreads) {
    float s = 0.f;
    for (uint32_t i = 0; i < cl; ++i) s += ld_dsmem(mapa_shared(base + e * 4, i));
    emit(e / W, e % W, s);
  }
  cluster_sync_all();
}

template <int DT, int TPR>
__global__ void __launch_bounds__(kXThreads) xattn_fwd_scalar(const XAttn a, int RB) {
  constexpr int DP = DT * TPR, LD = DP + 4;
  extern __shared__ __align__(16) float xsm[];
  float *sk = xsm, *sv = xsm + kXTile * LD;
  __shared__ uint8_t there[kXTile];
  const int KS = kXThreads / (RB * TPR);
  const int part = threadIdx.x % TPR, lr = (threadIdx.x / TPR) % RB, slice = threadIdx.x / (TPR * RB);
  const int b = blockIdx.z, n = blockIdx.y;
  const int cl = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
  const int rows = a.group * a.Tq;
  const int r0 = (blockIdx.x / cl) * RB, r = r0 + lr;
  const int g = r / a.Tq, t = r - g * a.Tq, h = n * a.group + g;
  const bool row_ok = r < rows;
  const int dims = a.d - part * DT;
  float q[DT], o[DT];
  load_row<DT>(static_cast<const float*>(a.q) + b * a.qs[0] + t * a.qs[1] + h * a.qs[2] + part * DT, dims, row_ok, q);
#pragma unroll
  for (int i = 0; i < DT; ++i) o[i] = 0.f;
  float m = -INFINITY, l = 0.f;
  const int keys = xattn_keys(a, b);
  const float* kb = static_cast<const float*>(a.k) + b * a.ks[0] + n * a.ks[2];
  const float* vb = static_cast<const float*>(a.v) + b * a.vs[0] + n * a.vs[2];
  const uint8_t* mask = a.key_mask == nullptr ? nullptr : a.key_mask + static_cast<int64_t>(b) * a.Tk;
  for (int j0 = rank * kXTile; j0 < keys; j0 += cl * kXTile) {
    const int nk = min(kXTile, keys - j0);
    auto ok = [&](int i) { return mask == nullptr || __ldg(mask + j0 + i) != 0; };
    __syncthreads();
    stage_rows<DP>(sk, nk, a.d, [&](int i) { return kb + (j0 + i) * a.ks[1]; }, ok);
    stage_rows<DP>(sv, nk, a.d, [&](int i) { return vb + (j0 + i) * a.vs[1]; }, ok);
    if (threadIdx.x < kXTile) there[threadIdx.x] = threadIdx.x < nk && ok(threadIdx.x);
    __syncthreads();
    for (int j = slice; j < kXTile; j += KS) {
      const float s = row_dot<DT, TPR>(q, sk + j * LD + part * DT) * a.c;
      if (!there[j]) continue;
      if (s > m) {
        const float f = ex2f(m - s);
        l *= f;
#pragma unroll
        for (int i = 0; i < DT; ++i) o[i] *= f;
        m = s;
      }
      const float p = s == -INFINITY ? 0.f : ex2f(s - m);  // a NaN logit stays one
      l += p;
      row_axpy<DT>(p, sv + j * LD + part * DT, o);
    }
  }
  // join the slices and blocks: rescale everybody's share to the common maximum first
  __syncthreads();
  float* ms = xsm;                       // [KS][RB]
  float* acc = xsm + kXThreads;          // [KS][RB][DP + 1]
  constexpr int W = DP + 1;
  if (part == 0) ms[slice * RB + lr] = m;
  __syncthreads();
  float top = -INFINITY;
  for (int i = 0; i < KS; ++i) top = fmaxf(top, ms[i * RB + lr]);
  if (cl > 1) {
    __syncthreads();
    if (part == 0 && slice == 0) ms[lr] = top;
    cluster_sync_all();
    const uint32_t at = smem_u32(ms + lr);
    for (int i = 0; i < cl; ++i) top = fmaxf(top, ld_dsmem(mapa_shared(at, i)));
  }
  const float f = m == -INFINITY ? 0.f : ex2f(m - top);
  float* mine = acc + (slice * RB + lr) * W;
#pragma unroll
  for (int i = 0; i < DT; ++i) mine[part * DT + i] = o[i] * f;
  if (part == 0) mine[DP] = l * f;
  // the sums, then the division: the row's denominator is summed with its entries
  __syncthreads();
  const int ne = RB * W;
  for (int e = threadIdx.x; e < ne; e += kXThreads) {
    float s = acc[e];
    for (int i = 1; i < KS; ++i) s += acc[i * ne + e];
    acc[e] = s;
  }
  if (cl > 1) cluster_sync_all(); else __syncthreads();
  const uint32_t abase = smem_u32(acc), mbase = smem_u32(ms);
  for (int e = rank * kXThreads + threadIdx.x; e < ne; e += cl * kXThreads) {
    const int er = e / W, col = e % W, rr = r0 + er;
    float s = 0.f, den = 0.f;
    if (cl == 1) {
      s = acc[e], den = acc[er * W + DP];
    } else {
      for (int i = 0; i < cl; ++i) {
        s += ld_dsmem(mapa_shared(abase + e * 4, i));
        den += ld_dsmem(mapa_shared(abase + (er * W + DP) * 4, i));
      }
    }
    if (rr >= rows) continue;
    const int eg = rr / a.Tq, et = rr - eg * a.Tq, eh = n * a.group + eg;
    if (col == DP) {
      if (a.lse != nullptr) {
        float mm = ms[er];
        if (cl > 1) {
          for (int i = 0; i < cl; ++i) mm = fmaxf(mm, ld_dsmem(mapa_shared(mbase + er * 4, i)));
        } else {
          for (int i = 1; i < KS; ++i) mm = fmaxf(mm, ms[i * RB + er]);
        }
        a.lse[(static_cast<int64_t>(b) * a.heads + eh) * a.Tq + et] = den > 0.f ? mm + log2f(den) : INFINITY;
      }
    } else if (col < a.d) {
      const float y = den > 0.f ? s / den : (den == 0.f ? 0.f : s / den);
      *(static_cast<float*>(a.out) + b * a.os[0] + et * a.os[1] + eh * a.os[2] + col) = y;
      if (a.out_f32 != nullptr)
        a.out_f32[((static_cast<int64_t>(b) * a.Tq + et) * a.heads + eh) * a.d + col] = y;
    }
  }
  if (cl > 1) cluster_sync_all();
}

// dQ: the forward's loop with p from the saved statistics. Also writes D for the dK / dV kernel.
template <int DT, int TPR>
__global__ void __launch_bounds__(kXThreads) xattn_dq_scalar(const XAttn a, int RB) {
  constexpr int DP = DT * TPR, LD = DP + 4;
  extern __shared__ __align__(16) float xsm[];
  float *sk = xsm, *sv = xsm + kXTile * LD;
  __shared__ uint8_t there[kXTile];
  const int KS = kXThreads / (RB * TPR);
  const int part = threadIdx.x % TPR, lr = (threadIdx.x / TPR) % RB, slice = threadIdx.x / (TPR * RB);
  const int b = blockIdx.z, n = blockIdx.y;
  const int cl = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
  const int rows = a.group * a.Tq;
  const int r0 = (blockIdx.x / cl) * RB, r = r0 + lr;
  const int g = r / a.Tq, t = r - g * a.Tq, h = n * a.group + g;
  const bool row_ok = r < rows;
  const int dims = a.d - part * DT;
  float q[DT], dO[DT], dq[DT];
  load_row<DT>(static_cast<const float*>(a.q) + b * a.qs[0] + t * a.qs[1] + h * a.qs[2] + part * DT, dims, row_ok, q);
  load_row<DT>(static_cast<const float*>(a.dout) + b * a.os[0] + t * a.os[1] + h * a.os[2] + part * DT, dims, row_ok,
                  dO);
  const int64_t stat = (static_cast<int64_t>(b) * a.heads + h) * a.Tq + t;
  // D in the order of dP's sum, so that a row with one key has dP - D = 0 exactly
  load_row<DT>(a.out_f32 + ((static_cast<int64_t>(b) * a.Tq + t) * a.heads + h) * a.d + part * DT, dims, row_ok,
                      dq);
  float delta = 0.f;
#pragma unroll
  for (int i = 0; i < DT; ++i) delta = fmaf(dO[i], dq[i], delta);
#pragma unroll
  for (int o = 1; o < TPR; o <<= 1) delta += __shfl_xor_sync(0xffffffffu, delta, o);
  const float lse = row_ok ? a.lse[stat] : INFINITY;
  if (row_ok && part == 0 && slice == 0 && rank == 0) a.delta[stat] = delta;
#pragma unroll
  for (int i = 0; i < DT; ++i) dq[i] = 0.f;
  if (a.dq != nullptr) {
    const int keys = xattn_keys(a, b);
    const float* kb = static_cast<const float*>(a.k) + b * a.ks[0] + n * a.ks[2];
    const float* vb = static_cast<const float*>(a.v) + b * a.vs[0] + n * a.vs[2];
    const uint8_t* mask = a.key_mask == nullptr ? nullptr : a.key_mask + static_cast<int64_t>(b) * a.Tk;
    for (int j0 = rank * kXTile; j0 < keys; j0 += cl * kXTile) {
      const int nk = min(kXTile, keys - j0);
      auto ok = [&](int i) { return mask == nullptr || __ldg(mask + j0 + i) != 0; };
      __syncthreads();
      stage_rows<DP>(sk, nk, a.d, [&](int i) { return kb + (j0 + i) * a.ks[1]; }, ok);
      stage_rows<DP>(sv, nk, a.d, [&](int i) { return vb + (j0 + i) * a.vs[1]; }, ok);
      if (threadIdx.x < kXTile) there[threadIdx.x] = threadIdx.x < nk && ok(threadIdx.x);
      __syncthreads();
      for (int j = slice; j < kXTile; j += KS) {
        const float s = row_dot<DT, TPR>(q, sk + j * LD + part * DT) * a.c;
        const float dp = row_dot<DT, TPR>(dO, sv + j * LD + part * DT);
        if (!there[j]) continue;
        row_axpy<DT>(ex2f(s - lse) * (dp - delta), sk + j * LD + part * DT, dq);
      }
    }
    __syncthreads();
    float* mine = xsm + (slice * RB + lr) * DP + part * DT;
#pragma unroll
    for (int i = 0; i < DT; ++i) mine[i] = dq[i];
    merge_sums(xsm, KS, RB, DP, [&](int er, int col, float s) {
      const int rr = r0 + er;
      if (rr >= rows || col >= a.d) return;
      const int eg = rr / a.Tq, et = rr - eg * a.Tq, eh = n * a.group + eg;
      *(static_cast<float*>(a.dq) + ((static_cast<int64_t>(b) * a.Tq + et) * a.heads + eh) * a.d + col) = s * a.scale;
    });
  }
}

// dK, dV: a thread owns (part of) one key; the block's slices walk the query rows.
template <int DT, int TPR>
__global__ void __launch_bounds__(kXThreads) xattn_dkv_scalar(const XAttn a, int RB) {
  constexpr int DP = DT * TPR, LD = DP + 4;
  extern __shared__ __align__(16) float xsm[];
  float *sq = xsm, *so = xsm + kXTile * LD;
  __shared__ float s_lse[kXTile], s_delta[kXTile];
  const int KS = kXThreads / (RB * TPR);
  const int part = threadIdx.x % TPR, lr = (threadIdx.x / TPR) % RB, slice = threadIdx.x / (TPR * RB);
  const int b = blockIdx.z, n = blockIdx.y;
  const int cl = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
  const int rows = a.group * a.Tq;
  const int j0 = (blockIdx.x / cl) * RB, j = j0 + lr;
  const bool key_ok = j < xattn_keys(a, b) &&
                      (a.key_mask == nullptr || __ldg(a.key_mask + static_cast<int64_t>(b) * a.Tk + j) != 0);
  const int dims = a.d - part * DT;
  float k[DT], v[DT], dk[DT], dv[DT];
  load_row<DT>(static_cast<const float*>(a.k) + b * a.ks[0] + j * a.ks[1] + n * a.ks[2] + part * DT, dims, key_ok, k);
  load_row<DT>(static_cast<const float*>(a.v) + b * a.vs[0] + j * a.vs[1] + n * a.vs[2] + part * DT, dims, key_ok, v);
#pragma unroll
  for (int i = 0; i < DT; ++i) dk[i] = 0.f, dv[i] = 0.f;
  for (int r0 = rank * kXTile; r0 < rows; r0 += cl * kXTile) {
    const int nr = min(kXTile, rows - r0);
    auto at = [&](int i, const int64_t (&st)[3]) {
      const int r = r0 + i, g = r / a.Tq, t = r - g * a.Tq;
      return b * st[0] + t * st[1] + (n * a.group + g) * st[2];
    };
    auto ok = [](int) { return true; };
    __syncthreads();
    stage_rows<DP>(sq, nr, a.d, [&](int i) { return static_cast<const float*>(a.q) + at(i, a.qs); }, ok);
    stage_rows<DP>(so, nr, a.d, [&](int i) { return static_cast<const float*>(a.dout) + at(i, a.os); }, ok);
    if (threadIdx.x < kXTile) {
      const int i = threadIdx.x, r = r0 + i, g = r / a.Tq, t = r - g * a.Tq;
      const int64_t stat = (static_cast<int64_t>(b) * a.heads + n * a.group + g) * a.Tq + t;
      s_lse[i] = i < nr ? a.lse[stat] : INFINITY;
      s_delta[i] = i < nr ? a.delta[stat] : 0.f;
    }
    __syncthreads();
    for (int i = slice; i < kXTile; i += KS) {
      const float s = row_dot<DT, TPR>(k, sq + i * LD + part * DT) * a.c;
      const float dp = row_dot<DT, TPR>(v, so + i * LD + part * DT);
      if (!key_ok || i >= nr) continue;
      const float p = ex2f(s - s_lse[i]);
      row_axpy<DT>(p, so + i * LD + part * DT, dv);
      row_axpy<DT>(p * (dp - s_delta[i]), sq + i * LD + part * DT, dk);
    }
  }
  __syncthreads();
  float* mine = xsm + (slice * RB + lr) * (2 * DP) + part * DT;
#pragma unroll
  for (int i = 0; i < DT; ++i) mine[i] = dk[i], mine[DP + i] = dv[i];
  merge_sums(xsm, KS, RB, 2 * DP, [&](int er, int col, float s) {
    const int jj = j0 + er, c = col % DP;
    if (jj >= a.Tk || c >= a.d) return;
    const int64_t to = ((static_cast<int64_t>(b) * a.Tk + jj) * a.kv_heads + n) * a.d + c;
    if (col < DP)
      *(static_cast<float*>(a.dk) + to) = s * a.scale;
    else
      *(static_cast<float*>(a.dv) + to) = s;
  });
}

// Launch
// Rows per block (a power of two, at most 128 / tpr) and blocks per cluster for `own` rows that
// each walk `other` entries: blocks are added along `other` until the device is filled.
static void xattn_plan(int own, int other, int64_t pairs, int tpr, int* rb, int* cluster) {
  int r = 4;
  while (r < own && r < kXThreads / tpr) r *= 2;
  const int64_t blocks = pairs * ((own + r - 1) / r);
  int c = 1;
  while (c < 8 && blocks * c < 2 * 148 && other > c * kXTile) c *= 2;
  *rb = r;
  *cluster = c;
}

template <int DT, int TPR>
static int xattn_scalar(const XAttn& a, bool backward, cudaStream_t stream) {
  constexpr int DP = DT * TPR;
  const size_t tiles = 2 * kXTile * (DP + 4) * sizeof(float);
  const int64_t pairs = static_cast<int64_t>(a.B) * a.kv_heads;
  const int rows = a.group * a.Tq;
  int rb, cl;
  if (!backward) {
    xattn_plan(rows, a.Tk, pairs, TPR, &rb, &cl);
    const size_t merge = (kXThreads + kXThreads / TPR * (DP + 1)) * sizeof(float);
    return launch_cluster(xattn_fwd_scalar<DT, TPR>, dim3((rows + rb - 1) / rb * cl, a.kv_heads, a.B), kXThreads,
                          tiles > merge ? tiles : merge, cl, stream, a, rb);
  }
  xattn_plan(rows, a.Tk, pairs, TPR, &rb, &cl);
  size_t merge = kXThreads / TPR * DP * sizeof(float);
  int st = launch_cluster(xattn_dq_scalar<DT, TPR>, dim3((rows + rb - 1) / rb * cl, a.kv_heads, a.B), kXThreads,
                          tiles > merge ? tiles : merge, cl, stream, a, rb);
  if (st != SSAM_OK || a.dk == nullptr) return st;
  xattn_plan(a.Tk, rows, pairs, TPR, &rb, &cl);
  merge = kXThreads / TPR * 2 * DP * sizeof(float);
  return launch_cluster(xattn_dkv_scalar<DT, TPR>, dim3((a.Tk + rb - 1) / rb * cl, a.kv_heads, a.B), kXThreads,
                        tiles > merge ? tiles : merge, cl, stream, a, rb);
}

static int xattn_dispatch(const XAttn& a, int dtype, bool backward, cudaStream_t stream) {
  if (dtype == 0) return xattn_mma<__half>(a, backward, stream);
  if (dtype == 1) return xattn_mma<__nv_bfloat16>(a, backward, stream);
  if (a.d <= 16) return xattn_scalar<16, 1>(a, backward, stream);
  if (a.d <= 32) return xattn_scalar<32, 1>(a, backward, stream);
  if (a.d <= 64) return xattn_scalar<32, 2>(a, backward, stream);
  return xattn_scalar<32, 4>(a, backward, stream);
}

// Checks shared by both directions; the strides and pointers are those the kernels read with
// 16-byte (fp32: 16-byte, half: 8-byte and wider) vector loads.
static int xattn_check(const XAttn& a, int dtype) {
  if (a.B <= 0 || a.Tq <= 0 || a.Tk <= 0 || a.heads <= 0 || a.kv_heads <= 0 || a.d <= 0) return SSAM_ERR_INVALID;
  if (dtype < 0 || dtype > 2 || a.heads % a.kv_heads) return SSAM_ERR_INVALID;
  if (!(a.scale > 0.f) || a.scale > 3.0e38f) return SSAM_ERR_INVALID;
  if (a.d > 128 || a.d % 8 || a.B > 65535 || a.kv_heads > 65535) return SSAM_ERR_UNSUPPORTED;
  if (static_cast<int64_t>(a.group) * a.Tq > (1 << 30) || a.Tk > (1 << 30)) return SSAM_ERR_UNSUPPORTED;
  const int64_t unit = dtype == 2 ? 4 : 8;
  for (int i = 0; i < 3; ++i)
    if (a.qs[i] % unit || a.ks[i] % unit || a.vs[i] % unit || a.os[i] % unit) return SSAM_ERR_ALIGN;
  for (const void* p : {a.q, a.k, a.v})
    if (!aligned16(p)) return SSAM_ERR_ALIGN;
  return SSAM_OK;
}

static XAttn xattn_args(const void* q, const void* k, const void* v, const int64_t* s, int B, int Tq, int Tk, int heads,
                        int kv_heads, int d, float scale, const int32_t* key_lens, const uint8_t* key_mask) {
  XAttn a = {};
  a.q = q, a.k = k, a.v = v;
  for (int i = 0; i < 3; ++i) a.qs[i] = s[i], a.ks[i] = s[3 + i], a.vs[i] = s[6 + i], a.os[i] = s[9 + i];
  a.B = B, a.Tq = Tq, a.Tk = Tk, a.heads = heads, a.kv_heads = kv_heads, a.d = d;
  a.group = kv_heads > 0 ? heads / kv_heads : 0;
  a.scale = scale, a.c = scale * 1.4426950408889634f;
  a.key_lens = key_lens, a.key_mask = key_mask;
  return a;
}

int cross_attn_fwd(const void* q, const void* k, const void* v, const int64_t* strides, int B, int Tq, int Tk,
                   int heads, int kv_heads, int d, int dtype, float scale, const int32_t* key_lens,
                   const uint8_t* key_mask, void* out, float* out_f32, float* lse, cudaStream_t stream) {
  if (q == nullptr || k == nullptr || v == nullptr || out == nullptr || strides == nullptr) return SSAM_ERR_INVALID;
  XAttn a = xattn_args(q, k, v, strides, B, Tq, Tk, heads, kv_heads, d, scale, key_lens, key_mask);
  a.out = out, a.out_f32 = out_f32, a.lse = lse;
  const int st = xattn_check(a, dtype);
  if (st != SSAM_OK) return st;
  if (!aligned16(out) || (out_f32 != nullptr && !aligned16(out_f32))) return SSAM_ERR_ALIGN;
  return xattn_dispatch(a, dtype, false, stream);
}

int cross_attn_bwd_uses_stats(int Tk, int d, int dtype) { return xattn_uses_stats(Tk, d, dtype) ? 1 : 0; }

int cross_attn_bwd(const void* q, const void* k, const void* v, const void* dout, const int64_t* strides, int B, int Tq,
                   int Tk, int heads, int kv_heads, int d, int dtype, float scale, const int32_t* key_lens,
                   const uint8_t* key_mask, const float* out_f32, const float* lse, float* delta, void* dq, void* dk,
                   void* dv, cudaStream_t stream) {
  if (q == nullptr || k == nullptr || v == nullptr || dout == nullptr || strides == nullptr ||
      ((out_f32 == nullptr || lse == nullptr || delta == nullptr) && xattn_uses_stats(Tk, d, dtype)) ||
      (dk == nullptr) != (dv == nullptr))
    return SSAM_ERR_INVALID;
  XAttn a = xattn_args(q, k, v, strides, B, Tq, Tk, heads, kv_heads, d, scale, key_lens, key_mask);
  a.dout = dout, a.out_f32 = const_cast<float*>(out_f32), a.lse = const_cast<float*>(lse), a.delta = delta;
  a.dq = dq, a.dk = dk, a.dv = dv;
  const int st = xattn_check(a, dtype);
  if (st != SSAM_OK) return st;
  for (const void* p : {static_cast<const void*>(dout), static_cast<const void*>(out_f32),
                        static_cast<const void*>(dq), static_cast<const void*>(dk), static_cast<const void*>(dv)})
    if (!aligned16(p)) return SSAM_ERR_ALIGN;
  if (dq == nullptr && dk == nullptr) return SSAM_OK;
  return xattn_dispatch(a, dtype, true, stream);
}

}  // namespace ssam
