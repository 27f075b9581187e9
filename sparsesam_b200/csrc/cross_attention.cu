// Cross attention: the entry points and the fp32 kernels (formulas and conventions in cross_attention.cuh).
#include "cross_attention.cuh"

namespace ssam {

// ---------------------------------------------------------------------------
// fp32 inputs: scalar kernels (fp32 FMAs). A thread owns DT dims of one row, TPR threads share
// a row. A block holds RB rows x KS slices of the other axis (RB * KS * TPR = 128).
// ---------------------------------------------------------------------------
constexpr int kXThreads = 128;
// entries of the other axis staged at a time (two stages, filled by cp.async)
template <int DP>
constexpr int kXTile = DP == 16 ? 128 : DP == 32 ? 64 : DP == 64 ? 32 : 16;
template <int DP>
constexpr size_t kXStages = 2 * 2 * kXTile<DP> * (DP + 4) * sizeof(float);

// <a, b> in two chains of packed FMAs; every dot product of these kernels has this order, so that with one
// key dP and D are the same number.
template <int DT, int TPR, class B>
__device__ __forceinline__ float row_dot(const float2 (&a)[DT / 2], B b) {
  float2 s0 = make_float2(0.f, 0.f), s1 = s0;
#pragma unroll
  for (int i = 0; i < DT / 2; i += 2) {
    const float4 v = b(i / 2);
    s0 = fma2(a[i], make_float2(v.x, v.y), s0);
    s1 = fma2(a[i + 1], make_float2(v.z, v.w), s1);
  }
  s0 = add2(s0, s1);
  float s = s0.x + s0.y;
#pragma unroll
  for (int o = 1; o < TPR; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}
template <int DT, int TPR>
__device__ __forceinline__ float row_dot(const float2 (&a)[DT / 2], const float* b) {
  return row_dot<DT, TPR>(a, [b](int i) { return *reinterpret_cast<const float4*>(b + 4 * i); });
}
// the same for NR rows: b is read once
template <int DT, int TPR, int NR>
__device__ __forceinline__ void rows_dot(const float2 (&a)[NR][DT / 2], const float* b, float (&y)[NR]) {
  float2 s0[NR], s1[NR];
#pragma unroll
  for (int z = 0; z < NR; ++z) s0[z] = s1[z] = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < DT / 2; i += 2) {
    const float4 v = *reinterpret_cast<const float4*>(b + 2 * i);
#pragma unroll
    for (int z = 0; z < NR; ++z) {
      s0[z] = fma2(a[z][i], make_float2(v.x, v.y), s0[z]);
      s1[z] = fma2(a[z][i + 1], make_float2(v.z, v.w), s1[z]);
    }
  }
#pragma unroll
  for (int z = 0; z < NR; ++z) {
    s0[z] = add2(s0[z], s1[z]);
    y[z] = s0[z].x + s0[z].y;
#pragma unroll
    for (int o = 1; o < TPR; o <<= 1) y[z] += __shfl_xor_sync(0xffffffffu, y[z], o);
  }
}
template <int DT, int NR>
__device__ __forceinline__ void rows_axpy(const float (&w)[NR], const float* b, float2 (&acc)[NR][DT / 2]) {
#pragma unroll
  for (int i = 0; i < DT / 2; i += 2) {
    const float4 v = *reinterpret_cast<const float4*>(b + 2 * i);
#pragma unroll
    for (int z = 0; z < NR; ++z) {
      acc[z][i] = fma2(make_float2(w[z], w[z]), make_float2(v.x, v.y), acc[z][i]);
      acc[z][i + 1] = fma2(make_float2(w[z], w[z]), make_float2(v.z, v.w), acc[z][i + 1]);
    }
  }
}
template <int DT>
__device__ __forceinline__ void row_axpy(float w, const float* b, float2 (&acc)[DT / 2]) {
  const float2 w2 = make_float2(w, w);
#pragma unroll
  for (int i = 0; i < DT / 2; i += 2) {
    const float4 v = *reinterpret_cast<const float4*>(b + 2 * i);
    acc[i] = fma2(w2, make_float2(v.x, v.y), acc[i]);
    acc[i + 1] = fma2(w2, make_float2(v.z, v.w), acc[i + 1]);
  }
}
template <int DT>
__device__ __forceinline__ void load_row(const float* p, int dims, bool ok, float2 (&r)[DT / 2]) {
#pragma unroll
  for (int i = 0; i < DT; i += 4) {
    const float4 v = ok && i < dims ? __ldg(reinterpret_cast<const float4*>(p + i)) : make_float4(0.f, 0.f, 0.f, 0.f);
    r[i / 2] = make_float2(v.x, v.y), r[i / 2 + 1] = make_float2(v.z, v.w);
  }
}
template <int DT>
__device__ __forceinline__ void clear_row(float2 (&r)[DT / 2]) {
#pragma unroll
  for (int i = 0; i < DT / 2; ++i) r[i] = make_float2(0.f, 0.f);
}

// Starts the copy of `n` rows of width d into sm[kXTile][DP + 4]; rows n .. upto - 1, rows for which ok(i) is
// false, and channels past d, are zeros.
template <int DP, class P, class O>
__device__ __forceinline__ void stage_rows(float* sm, int n, int upto, int d, P row, O ok) {
  constexpr int V = DP / 4, LD = DP + 4;
#pragma unroll
  for (int e0 = 0; e0 < kXTile<DP> * V; e0 += kXThreads) {
    if (e0 >= upto * V) break;
    const int e = e0 + threadIdx.x, i = e / V, c = (e % V) * 4;
    const bool there = i < n && c < d && ok(i);
    cp_async16(smem_u32(sm + i * LD + c), there ? row(i) + c : row(0), there ? 16u : 0u);
  }
}
__device__ __forceinline__ void stage_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void stage_wait() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }

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

// The block's own rows, which lie heads * d apart, through shared memory: four lanes fetch a row's 64 bytes and more
// together, where a thread that reads its own row by itself touches 32 lines per load (image -> tokens, fp32, 64
// images: 144 us that way, 128 through shared memory). row(i) is row i's address, nullptr behind the last.
template <int DP, class R>
__device__ __forceinline__ void fetch_own(float* sm, int RB, int d, R row) {
  constexpr int V = DP / 4, LD = DP + 4;
  for (int e = threadIdx.x; e < RB * V; e += kXThreads) {
    const int i = e / V, c = e % V * 4;
    const float* p = row(i);
    const bool there = p != nullptr && c < d;
    cp_async16(smem_u32(sm + i * LD + c), there ? p + c : row(0), there ? 16u : 0u);
  }
}
template <int DT>
__device__ __forceinline__ void own_row(const float* p, float2 (&r)[DT / 2]) {
#pragma unroll
  for (int i = 0; i < DT; i += 4) {
    const float4 v = *reinterpret_cast<const float4*>(p + i);
    r[i / 2] = make_float2(v.x, v.y), r[i / 2 + 1] = make_float2(v.z, v.w);
  }
}
template <int DT>
__device__ __forceinline__ void put_row(float* p, const float2 (&r)[DT / 2], float f) {
#pragma unroll
  for (int i = 0; i < DT; i += 4)
    *reinterpret_cast<float4*>(p + i) = make_float4(r[i / 2].x * f, r[i / 2].y * f, r[i / 2 + 1].x * f, r[i / 2 + 1].y * f);
}

// What the two row kernels share: a block's place, and the walk over its keys. body(tile of K, tile of V, keys of
// the tile rounded up to the slices, their biases: 0, or -infinity where there is no key) is called with the tile in
// shared memory. False: every key that the block walked is masked, and its sums are to be left out (those of a query
// that is not finite are not 0).
struct XPlace {
  int part, lr, slice, KS, b, n, cl, rank, rows, r0, r, t, h;
  bool row_ok;
  // address of the block's row i in a tensor of queries, nullptr behind the last
  __device__ __forceinline__ const float* row_of(const XAttn& a, const float* p, const int64_t (&st)[3], int i) const {
    const int rr = r0 + i, gg = a.group == 1 ? 0 : rr / a.Tq, tt = rr - gg * a.Tq;
    return rr < rows ? p + b * st[0] + tt * st[1] + (n * a.group + gg) * st[2] : nullptr;
  }
  __device__ __forceinline__ XPlace(const XAttn& a, int RB, int TPR, int NR = 1) {
    KS = kXThreads / (RB * TPR);
    part = threadIdx.x % TPR, lr = threadIdx.x / TPR % RB, slice = threadIdx.x / (TPR * RB);
    b = blockIdx.z, n = blockIdx.y;
    cl = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
    rows = a.group * a.Tq;
    r0 = static_cast<int>(blockIdx.x) / cl * RB * NR, r = r0 + lr;
    const int g = r / a.Tq;
    t = r - g * a.Tq, h = n * a.group + g;
    row_ok = r < rows;
  }
};
template <int DP, class B>
__device__ __forceinline__ bool walk_keys(const XAttn& a, const XPlace& x, float* xsm, float (&bias)[2][kXTile<DP>], B body) {
  constexpr int XT = kXTile<DP>, LD = DP + 4;
  const int keys = xattn_keys(a, x.b);
  const float* kb = static_cast<const float*>(a.k) + x.b * a.ks[0] + x.n * a.ks[2];
  const float* vb = static_cast<const float*>(a.v) + x.b * a.vs[0] + x.n * a.vs[2];
  const uint8_t* mask = a.key_mask == nullptr ? nullptr : a.key_mask + static_cast<int64_t>(x.b) * a.Tk;
  bool some = false;
  auto stage = [&](int j0, int buf) {
    if (j0 < keys) {
      const int nk = min(XT, keys - j0), upto = (nk + x.KS - 1) / x.KS * x.KS;
      auto ok = [&](int i) { return mask == nullptr || __ldg(mask + j0 + i) != 0; };
      float* to = xsm + buf * 2 * XT * LD;
      stage_rows<DP>(to, nk, upto, a.d, [&](int i) { return kb + (j0 + i) * a.ks[1]; }, ok);
      stage_rows<DP>(to + XT * LD, nk, upto, a.d, [&](int i) { return vb + (j0 + i) * a.vs[1]; }, ok);
      if (threadIdx.x < XT) {
        const bool there = threadIdx.x < nk && ok(threadIdx.x);
        bias[buf][threadIdx.x] = there ? 0.f : -INFINITY;
        some |= there;
      }
    }
    stage_commit();
  };
  stage(x.rank * XT, 0);
  int buf = 0;
  for (int j0 = x.rank * XT; j0 < keys; j0 += x.cl * XT, buf ^= 1) {
    stage(j0 + x.cl * XT, buf ^ 1);
    stage_wait();
    __syncthreads();
    const float* sk = xsm + buf * 2 * XT * LD;
    body(sk, sk + XT * LD, (min(XT, keys - j0) + x.KS - 1) / x.KS * x.KS, bias[buf]);
    __syncthreads();                         // the other buffer is filled next
  }
  return mask == nullptr || __syncthreads_or(some);
}

// Joins the slices' and blocks' shares of the rows.
template <int DT, int TPR>
__device__ __forceinline__ void xattn_fwd_join(const XAttn& a, const XPlace& x, float* xsm, int RB, const float2 (&o)[DT / 2], float m,
                                               float l) {
  constexpr int DP = DT * TPR;
  const int part = x.part, lr = x.lr, slice = x.slice, KS = x.KS, b = x.b, n = x.n, cl = x.cl, rank = x.rank, rows = x.rows,
            r0 = x.r0;
  // rescale everybody's share to the common maximum first
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
  for (int i = 0; i < DT / 2; ++i) mine[part * DT + 2 * i] = o[i].x * f, mine[part * DT + 2 * i + 1] = o[i].y * f;
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

// NR rows to a thread, RB apart: K and V come out of shared memory once for all of them, which is what the kernel waits
// for (1024 x 1024, 16 x 8 heads of 16: 400 us with one row, 312 with two, of 64: 2040 and 1345; 4096 queries on 8
// keys, 64 x 8 heads of 16: 128 and 103, at 2.6 TB/s). NR > 1: one slice, no cluster.
// (The bounds are the blocks that fit anyway: 168 registers for NR 2, DT 32. Left to itself the compiler once took 196,
// and 4096 x 30 of 32 channels 113 us instead of 97.)
template <int DT, int TPR, int NR>
__global__ void __launch_bounds__(kXThreads, DT == 16 ? (NR == 1 ? 7 : 4) : (NR == 1 ? 4 : 3)) xattn_fwd_scalar(const XAttn args, int RB) {
  const XAttn a = follow(args, false);
  constexpr int DP = DT * TPR, LD = DP + 4, U = 4;
  extern __shared__ __align__(16) float xsm[];
  __shared__ float bias[2][kXTile<DP>];
  const XPlace x(a, RB, TPR, NR);
  const int part = x.part, lr = x.lr, slice = x.slice, KS = x.KS, b = x.b, n = x.n, cl = x.cl, rows = x.rows;
  float2 q[NR][DT / 2], o[NR][DT / 2];
  fetch_own<DP>(xsm, NR * RB, a.d, [&](int i) { return x.row_of(a, static_cast<const float*>(a.q), a.qs, i); });
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  float m[NR], l[NR];
#pragma unroll
  for (int z = 0; z < NR; ++z) {
    own_row<DT>(xsm + (z * RB + lr) * LD + part * DT, q[z]);
    clear_row<DT>(o[z]);
    m[z] = -INFINITY, l[z] = 0.f;
  }
  __syncthreads();
  const bool some = walk_keys<DP>(a, x, xsm, bias, [&](const float* sk, const float* sv, int nk, const float* here) {
    for (int j = slice; j < nk; j += U * KS) {           // U keys at a time: one look at the maximum
      float s[NR][U], top[NR];
#pragma unroll
      for (int z = 0; z < NR; ++z) top[z] = m[z];
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int z = 0; z < NR; ++z) s[z][u] = -INFINITY;
        if (j - slice + u * KS < nk) {                   // the same for all threads
          const int i = j + u * KS;
          float y[NR];
          rows_dot<DT, TPR, NR>(q, sk + i * LD + part * DT, y);
#pragma unroll
          for (int z = 0; z < NR; ++z) s[z][u] = fmaf(y[z], a.c, here[i]);   // -infinity: no such key
        }
#pragma unroll
        for (int z = 0; z < NR; ++z) top[z] = fmaxf(top[z], s[z][u]);
      }
#pragma unroll
      for (int z = 0; z < NR; ++z)
        if (top[z] > m[z]) {
          const float f = ex2f(m[z] - top[z]);
          l[z] *= f;
#pragma unroll
          for (int i = 0; i < DT / 2; ++i) o[z][i] = mul2(o[z][i], make_float2(f, f));
          m[z] = top[z];
        }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (j - slice + u * KS >= nk) break;
        float p[NR];
#pragma unroll
        for (int z = 0; z < NR; ++z) {
          p[z] = s[z][u] == -INFINITY ? 0.f : ex2f(s[z][u] - m[z]);  // a NaN logit stays one
          l[z] += p[z];
        }
        rows_axpy<DT, NR>(p, sv + (j + u * KS) * LD + part * DT, o);
      }
    }
  });
  if (!some) {
#pragma unroll
    for (int z = 0; z < NR; ++z) clear_row<DT>(o[z]), m[z] = -INFINITY, l[z] = 0.f;
  }
  if (NR > 1 || (KS == 1 && cl == 1)) {      // a row is one group of TPR threads: out through shared memory, as it came
#pragma unroll
    for (int z = 0; z < NR; ++z) {
      const float inv = l[z] == 0.f ? 0.f : 1.f / l[z];
      put_row<DT>(xsm + (z * RB + lr) * LD + part * DT, o[z], inv);
      const int r = x.r + z * RB;
      if (a.lse != nullptr && part == 0 && r < rows)
        a.lse[(static_cast<int64_t>(b) * a.heads + n * a.group) * a.Tq + r] = l[z] == 0.f ? INFINITY : m[z] + log2f(l[z]);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < NR * RB * (DP / 4); e += kXThreads) {
      const int i = e / (DP / 4), col = e % (DP / 4) * 4;
      float* to = const_cast<float*>(x.row_of(a, static_cast<const float*>(a.out), a.os, i));
      if (to == nullptr || col >= a.d) continue;
      const float4 y = *reinterpret_cast<const float4*>(xsm + i * LD + col);
      *reinterpret_cast<float4*>(to + col) = y;
      if (a.out_f32 != nullptr) {
        const int64_t dense[3] = {static_cast<int64_t>(a.Tq) * a.heads * a.d, static_cast<int64_t>(a.heads) * a.d, a.d};
        *reinterpret_cast<float4*>(const_cast<float*>(x.row_of(a, a.out_f32, dense, i)) + col) = y;
      }
    }
    return;
  }
  if constexpr (NR == 1) xattn_fwd_join<DT, TPR>(a, x, xsm, RB, o[0], m[0], l[0]);
}

// dQ: the forward's loop with p from the saved statistics. Also writes D for the dK / dV kernel.
template <int DT, int TPR>
__global__ void __launch_bounds__(kXThreads) xattn_dq_scalar(const XAttn args, int RB) {
  const XAttn a = follow(args, false);
  constexpr int DP = DT * TPR, LD = DP + 4;
  extern __shared__ __align__(16) float xsm[];
  __shared__ float bias[2][kXTile<DP>];
  const XPlace x(a, RB, TPR);
  const int part = x.part, slice = x.slice, KS = x.KS, b = x.b;
  float2 q[DT / 2], dO[DT / 2], dq[DT / 2];
  const int64_t stat = (static_cast<int64_t>(b) * a.heads + x.h) * a.Tq + x.t;
  const int64_t dense[3] = {static_cast<int64_t>(a.Tq) * a.heads * a.d, static_cast<int64_t>(a.heads) * a.d, a.d};
  const int own = RB * LD;
  fetch_own<DP>(xsm, RB, a.d, [&](int i) { return x.row_of(a, static_cast<const float*>(a.q), a.qs, i); });
  fetch_own<DP>(xsm + own, RB, a.d, [&](int i) { return x.row_of(a, static_cast<const float*>(a.dout), a.os, i); });
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  own_row<DT>(xsm + x.lr * LD + part * DT, q);
  own_row<DT>(xsm + own + x.lr * LD + part * DT, dO);
  __syncthreads();
  fetch_own<DP>(xsm, RB, a.d, [&](int i) { return x.row_of(a, a.out_f32, dense, i); });
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  own_row<DT>(xsm + x.lr * LD + part * DT, dq);
  __syncthreads();
  const float delta = row_dot<DT, TPR>(dO, [&](int i) { return make_float4(dq[2 * i].x, dq[2 * i].y, dq[2 * i + 1].x, dq[2 * i + 1].y); });
  const float lse = x.row_ok ? a.lse[stat] : INFINITY;
  if (x.row_ok && part == 0 && slice == 0 && x.rank == 0) a.delta[stat] = delta;
  if (a.dq == nullptr) return;               // only D was wanted
  clear_row<DT>(dq);
  const bool some = walk_keys<DP>(a, x, xsm, bias, [&](const float* sk, const float* sv, int nk, const float* here) {
#pragma unroll 1
    for (int j = slice; j < nk; j += KS) {
      const float s = fmaf(row_dot<DT, TPR>(q, sk + j * LD + part * DT), a.c, here[j]);
      const float dp = row_dot<DT, TPR>(dO, sv + j * LD + part * DT);
      row_axpy<DT>(ex2f(s - lse) * (dp - delta), sk + j * LD + part * DT, dq);
    }
  });
  if (!some) clear_row<DT>(dq);
  if (KS == 1 && x.cl == 1) {
    put_row<DT>(xsm + x.lr * LD + part * DT, dq, a.scale);
    __syncthreads();
    for (int e = threadIdx.x; e < RB * (DP / 4); e += kXThreads) {
      const int i = e / (DP / 4), col = e % (DP / 4) * 4;
      float* to = const_cast<float*>(x.row_of(a, static_cast<const float*>(a.dq), dense, i));
      if (to != nullptr && col < a.d) *reinterpret_cast<float4*>(to + col) = *reinterpret_cast<const float4*>(xsm + i * LD + col);
    }
    return;
  }
  __syncthreads();
  float* mine = xsm + (slice * RB + x.lr) * DP + part * DT;
#pragma unroll
  for (int i = 0; i < DT / 2; ++i) mine[2 * i] = dq[i].x, mine[2 * i + 1] = dq[i].y;
  merge_sums(xsm, KS, RB, DP, [&](int er, int col, float s) {
    const int rr = x.r0 + er;
    if (rr >= x.rows || col >= a.d) return;
    const int eg = rr / a.Tq, et = rr - eg * a.Tq, eh = x.n * a.group + eg;
    static_cast<float*>(a.dq)[((static_cast<int64_t>(b) * a.Tq + et) * a.heads + eh) * a.d + col] = s * a.scale;
  });
}

// dK, dV: a thread owns (part of) one key; the block's slices walk the query rows.
template <int DT, int TPR>
__global__ void __launch_bounds__(kXThreads) xattn_dkv_scalar(const XAttn args, int RB) {
  const XAttn a = follow(args, false);
  constexpr int DP = DT * TPR, LD = DP + 4, XT = kXTile<DP>;
  extern __shared__ __align__(16) float xsm[];
  __shared__ float s_lse[2][XT], s_delta[2][XT];
  const int KS = kXThreads / (RB * TPR);
  const int part = threadIdx.x % TPR, lr = (threadIdx.x / TPR) % RB, slice = threadIdx.x / (TPR * RB);
  const int b = blockIdx.z, n = blockIdx.y;
  const int cl = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
  const int rows = a.group * a.Tq;
  const int j0 = (blockIdx.x / cl) * RB, j = j0 + lr;
  const bool key_ok = j < xattn_keys(a, b) &&
                      (a.key_mask == nullptr || __ldg(a.key_mask + static_cast<int64_t>(b) * a.Tk + j) != 0);
  const int dims = a.d - part * DT;
  float2 k[DT / 2], v[DT / 2], dk[DT / 2], dv[DT / 2];
  load_row<DT>(static_cast<const float*>(a.k) + b * a.ks[0] + j * a.ks[1] + n * a.ks[2] + part * DT, dims, key_ok, k);
  load_row<DT>(static_cast<const float*>(a.v) + b * a.vs[0] + j * a.vs[1] + n * a.vs[2] + part * DT, dims, key_ok, v);
  clear_row<DT>(dk);
  clear_row<DT>(dv);
  auto stage = [&](int r0, int buf) {
    if (r0 < rows) {
      const int nr = min(XT, rows - r0);
      auto at = [&](int i, const int64_t (&st)[3]) {
        const int r = r0 + i, g = a.group == 1 ? 0 : r / a.Tq, t = r - g * a.Tq;
        return b * st[0] + t * st[1] + (n * a.group + g) * st[2];
      };
      auto ok = [](int) { return true; };
      float* to = xsm + buf * 2 * XT * LD;
      const int upto = (nr + KS - 1) / KS * KS;
      stage_rows<DP>(to, nr, upto, a.d, [&](int i) { return static_cast<const float*>(a.q) + at(i, a.qs); }, ok);
      stage_rows<DP>(to + XT * LD, nr, upto, a.d, [&](int i) { return static_cast<const float*>(a.dout) + at(i, a.os); }, ok);
      const int64_t stat = (static_cast<int64_t>(b) * a.heads + n * a.group) * a.Tq + r0;   // rows of a key head follow one another
      if (threadIdx.x < XT) {
        s_lse[buf][threadIdx.x] = threadIdx.x < nr ? a.lse[stat + threadIdx.x] : INFINITY;
        s_delta[buf][threadIdx.x] = threadIdx.x < nr ? a.delta[stat + threadIdx.x] : 0.f;
      }
    }
    stage_commit();
  };
  stage(rank * XT, 0);
  int buf = 0;
  for (int r0 = rank * XT; r0 < rows; r0 += cl * XT, buf ^= 1) {
    stage(r0 + cl * XT, buf ^ 1);
    stage_wait();
    __syncthreads();
    const float *sq = xsm + buf * 2 * XT * LD, *so = sq + XT * LD;
    const int nr = (min(XT, rows - r0) + KS - 1) / KS * KS;      // entries behind the last have p = 2^-inf = 0
#pragma unroll 1
    for (int i = slice; i < nr; i += KS) {
      const float s = row_dot<DT, TPR>(k, sq + i * LD + part * DT) * a.c;
      const float dp = row_dot<DT, TPR>(v, so + i * LD + part * DT);
      const float p = key_ok ? ex2f(s - s_lse[buf][i]) : 0.f;
      row_axpy<DT>(p, so + i * LD + part * DT, dv);
      row_axpy<DT>(p * (dp - s_delta[buf][i]), sq + i * LD + part * DT, dk);
    }
    __syncthreads();
  }
  if (!key_ok) clear_row<DT>(dk), clear_row<DT>(dv);   // also where a query or its gradient is not finite
  __syncthreads();
  float* mine = xsm + (slice * RB + lr) * (2 * DP) + part * DT;
#pragma unroll
  for (int i = 0; i < DT / 2; ++i) {
    mine[2 * i] = dk[i].x, mine[2 * i + 1] = dk[i].y;
    mine[DP + 2 * i] = dv[i].x, mine[DP + 2 * i + 1] = dv[i].y;
  }
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
// Rows per block (a power of two, at most 128 / tpr: few rows left empty, and a block costs as much as 16 rows) and
// blocks per cluster for `own` rows that each walk `other` entries, `tile` at a time: blocks are added along `other`
// until the device has four of these small blocks per SM.
static void xattn_plan(int own, int other, int64_t pairs, int tpr, int tile, int* rb, int* cluster) {
  int r = kXThreads / tpr;
  for (int x = r / 2; x >= 4; x /= 2)
    if ((own + x - 1) / x * (x + 16) < (own + r - 1) / r * (r + 16)) r = x;
  const int64_t blocks = pairs * ((own + r - 1) / r);
  int c = 1;
  while (c < 8 && blocks * c < 4 * 148 && other > c * tile) c *= 2;
  *rb = r;
  *cluster = c;
}

template <int DT, int TPR>
static int xattn_scalar(const XAttn& a, bool backward, cudaStream_t stream) {
  constexpr int DP = DT * TPR, XT = kXTile<DP>;
  constexpr size_t stages = kXStages<DP>;
  const int64_t pairs = static_cast<int64_t>(a.B) * a.kv_heads;
  const int rows = a.group * a.Tq;
  int rb, cl;
  xattn_plan(rows, a.Tk, pairs, TPR, XT, &rb, &cl);
  const dim3 by_rows((rows + rb - 1) / rb * cl, a.kv_heads, a.B);
  if (!backward) {
    constexpr size_t merge = (kXThreads + kXThreads / TPR * (DP + 1)) * sizeof(float);
    static_assert(merge <= 48 << 10 && stages <= 48 << 10, "no opt-in needed");
    // two rows to a thread where that still leaves every SM two blocks (DT 32: four, of which three run at once; 512
    // blocks of 32 channels took 696 us where 1024 of one row took 586)
    const int two = (rows + 2 * rb - 1) / (2 * rb);
    static_assert(2 * kXThreads / TPR * (DP + 4) * sizeof(float) <= stages, "the block's own rows");
    if (rb * TPR == kXThreads && cl == 1 && rows > rb && pairs * two >= (DT == 16 ? 2 : 4) * 148)
      return launch_following(xattn_fwd_scalar<DT, TPR, 2>, dim3(two, a.kv_heads, a.B), kXThreads, stages, 1, stream, a, rb);
    return launch_following(xattn_fwd_scalar<DT, TPR, 1>, by_rows, kXThreads, stages > merge ? stages : merge, cl, stream, a, rb);
  }
  constexpr size_t merge = kXThreads / TPR * 2 * DP * sizeof(float);
  static_assert(merge <= 48 << 10, "no opt-in needed");
  const int st = launch_following(xattn_dq_scalar<DT, TPR>, by_rows, kXThreads, stages > merge ? stages : merge, cl, stream, a, rb);
  if (st != SSAM_OK || a.dk == nullptr) return st;
  xattn_plan(a.Tk, rows, pairs, TPR, XT, &rb, &cl);
  return launch_following(xattn_dkv_scalar<DT, TPR>, dim3((a.Tk + rb - 1) / rb * cl, a.kv_heads, a.B), kXThreads,
                        stages > merge ? stages : merge, cl, stream, a, rb);
}

static int xattn_dispatch(const XAttn& a, int dtype, bool backward, cudaStream_t stream) {
  if (dtype == 0) return xattn_fp16(a, backward, stream);
  if (dtype == 1) return xattn_bf16(a, backward, stream);
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
  if (!(a.scale > 0.f) || a.scale > 2.0e38f) return SSAM_ERR_INVALID;   // scale log2(e) is finite
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
