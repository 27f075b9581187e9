// Cross attention of two long sides on the 5th-generation tensor cores (formulas and conventions in
// cross_attention.cuh): heads of up to 64 channels (zero-padded to 64), fp16 / bf16 forward, bf16 backward.
//
// A block of 128 threads owns a tile of 128 entries of one side (a thread is an entry and a TMEM lane) and walks the
// other side 64 entries at a time:
//   S = X1 Y1^T (and dP = X2 Y2^T)      tcgen05.mma, both operands in shared memory, K-major, 128-byte swizzle
//   P (and dS) from S by its thread     tcgen05.ld, exponentials, tcgen05.st over the columns of S (and dP)
//   sums += P Y2, dS Y1                 tcgen05.mma with the first operand in TMEM; the same shared-memory tile now
//                                       MN-major (its rows are the k axis)
// P and dS enter as two half terms: of every 32 fp32 columns, the first 16 take the values, the others the remainders.
// The chain load -> mma -> softmax -> mma of a block is serial; 4 (forward: 128 TMEM columns) or 2 (backward: 256)
// blocks per SM run each other's gaps. Tiles come by cp.async rather than TMA: rows of masked keys and channels past
// d are zero-filled on the way, and any row stride will do. Where tiles leave the device empty, the other side is
// split over a cluster and joined through distributed shared memory in rank order.
// Every wait is bounded; a block whose wait ran out raises SSAM_ERR_TIMEOUT and leaves.
#include <cuda_fp16.h>

#include "common.cuh"
#include "cross_attention.cuh"
#include "host_util.h"

namespace ssam {

constexpr int kTcOwn = 128, kTcOther = 64, kTcThreads = 128;
constexpr int kTcTile = kTcOwn * 128, kTcStage = 2 * kTcOther * 128;    // bytes

// 16-byte chunk c (8 channels) of row r of a 128-byte-swizzled tile
__device__ __forceinline__ uint32_t tc_chunk(uint32_t tile, int r, int c) { return tile + r * 128 + ((c ^ (r & 7)) << 4); }

// Starts the copies of ROWS rows (row(i): address, nullptr: zeros) into a tile.
template <class T, int ROWS, class R>
__device__ __forceinline__ void tc_fetch(uint32_t tile, int d, const T* valid, R row) {
  const int c = threadIdx.x % 8;
#pragma unroll
  for (int i0 = 0; i0 < ROWS; i0 += kTcThreads / 8) {
    const int i = i0 + threadIdx.x / 8;
    const T* p = row(i);
    const bool there = p != nullptr && c * 8 < d;
    cp_async16(tc_chunk(tile, i, c), there ? p + c * 8 : valid, there ? 16u : 0u);
  }
}
template <class T>
constexpr uint32_t tc_idesc(uint32_t b_mn) {
  const uint32_t f = sizeof(T) == 2 && std::is_same<T, __half>::value ? 0u : 1u;
  return (1u << 4) | (f << 7) | (f << 10) | (b_mn << 16) | ((64u >> 3) << 17) | ((128u >> 4) << 24);
}
// D[128 x 64] = A[128 x 64 channels] B[64 entries x 64 channels]^T
template <class T>
__device__ __forceinline__ void tc_scores(uint32_t d_tmem, uint32_t a, uint32_t b) {
#pragma unroll
  for (int k = 0; k < 4; ++k)
    umma_f16_ss(d_tmem, make_smem_desc(a + k * 32, 16, 1024, kSw128), make_smem_desc(b + k * 32, 16, 1024, kSw128),
                tc_idesc<T>(0), k > 0);
}
// D[128 x 64 channels] (+)= P[128 x 64 entries] B[64 entries x 64 channels], P in TMEM as [16 values | 16 remainders] twice
template <class T>
__device__ __forceinline__ void tc_sums(uint32_t d_tmem, uint32_t p_tmem, uint32_t b, bool accumulate) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint64_t desc = make_smem_desc(b + k * 2048, 16, 1024, kSw128);
    const uint32_t p = p_tmem + (k / 2) * 32 + (k % 2) * 8;
    umma_f16_ts(d_tmem, p, desc, tc_idesc<T>(1), accumulate || k > 0);
    umma_f16_ts(d_tmem, p + 16, desc, tc_idesc<T>(1), 1u);
  }
}

template <class T>
__device__ __forceinline__ uint32_t tc_pack(float x, float y);
template <>
__device__ __forceinline__ uint32_t tc_pack<__nv_bfloat16>(float x, float y) { return pack_bf16x2(x, y); }
template <>
__device__ __forceinline__ uint32_t tc_pack<__half>(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <class T>
__device__ __forceinline__ float2 tc_unpack(uint32_t u) {
  if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&u));
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
// value pair -> out[i] (values), out[16 + i] (remainders)
template <class T>
__device__ __forceinline__ void tc_split(float2 p, uint32_t (&out)[32], int i) {
  out[i] = tc_pack<T>(p.x, p.y);
  const float2 h = tc_unpack<T>(out[i]), r = add2(p, make_float2(-h.x, -h.y));
  out[16 + i] = tc_pack<T>(r.x, r.y);
}
__device__ __forceinline__ float4 ld_dsmem4(uint32_t cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(cluster_addr)
               : "memory");
  return v;
}
// 16-byte chunk c (4 floats) of row r of the join's [128][64] fp32 tile
__device__ __forceinline__ uint32_t tc_join_chunk(uint32_t tile, int r, int c) { return tile + r * 256 + ((c ^ (r & 15)) << 4); }

__device__ __forceinline__ void tc_read64(uint32_t t_lane, float2 (&v)[32]) {
  uint32_t r[2][32];
  tmem_ld_32x32b_x32(t_lane, r[0]);
  tmem_ld_32x32b_x32(t_lane + 32, r[1]);
  tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < 32; ++i)
    v[i] = make_float2(__uint_as_float(r[i / 16][2 * (i % 16)]), __uint_as_float(r[i / 16][2 * (i % 16) + 1]));
}
// Puts a thread's 64 sums, times f, into the join's tile.
__device__ __forceinline__ void tc_put64(uint32_t tile, int r, const float2 (&v)[32], float f) {
#pragma unroll
  for (int c = 0; c < 16; ++c)
    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(tc_join_chunk(tile, r, c)), "f"(v[2 * c].x * f),
                 "f"(v[2 * c].y * f), "f"(v[2 * c + 1].x * f), "f"(v[2 * c + 1].y * f)
                 : "memory");
}
template <class T>
__device__ __forceinline__ void tc_store_row(T* to, int d, const float2 (&v)[32], float f) {
#pragma unroll
  for (int c = 0; c < 8; ++c)
    if (c * 8 < d)
      *reinterpret_cast<uint4*>(to + c * 8) =
          make_uint4(tc_pack<T>(v[4 * c].x * f, v[4 * c].y * f), tc_pack<T>(v[4 * c + 1].x * f, v[4 * c + 1].y * f),
                     tc_pack<T>(v[4 * c + 2].x * f, v[4 * c + 2].y * f), tc_pack<T>(v[4 * c + 3].x * f, v[4 * c + 3].y * f));
}

// What both kernels set up: barriers, TMEM, aligned shared memory.
struct TcBlock {
  uint32_t sm;          // 1024-byte aligned
  uint32_t tmem, t_lane;
  uint64_t* bars;       // [0] scores ready, [1] sums done
  __device__ __forceinline__ void open(uint8_t* raw, uint64_t* shared_bars, uint32_t* holder, uint32_t cols) {
    sm = (smem_u32(raw) + 1023u) & ~1023u;
    bars = shared_bars;
    if (threadIdx.x == 0) {
      mbar_init(&bars[0], 1);
      mbar_init(&bars[1], 1);
      fence_mbar_init();
    }
    if (threadIdx.x < 32) {
      tmem_alloc(holder, cols);
      tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    tmem = *holder;
    t_lane = tmem + (threadIdx.x / 32 * 32u << 16);
  }
  // Gives the TMEM back. Called before the blocks of a cluster wait for one another: a block that holds TMEM never
  // waits for one that may be waiting for some.
  __device__ __forceinline__ void close(uint32_t cols) const {
    cp_async_wait_all();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (threadIdx.x < 32) tmem_dealloc(tmem, cols);
  }
};
constexpr float kTcNone = -1e30f, kTcSlack = 8.f;

template <class T>
__global__ void __launch_bounds__(kTcThreads, 4) xattn_tc_fwd_kernel(const XAttn a) {
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t bars[2];
  __shared__ uint32_t holder;
  __shared__ __align__(16) float s_bias[2][kTcOther];
  __shared__ float s_ref[kTcOwn], s_l[kTcOwn];
  TcBlock B;
  B.open(raw, bars, &holder, 128);
  const uint32_t x1 = B.sm, ring = B.sm + kTcTile, tS = 0, tO = 64;
  const int tid = threadIdx.x;
  const int cl = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
  const int own0 = static_cast<int>(blockIdx.x) / cl * kTcOwn, h = blockIdx.y, b = blockIdx.z, n = h / a.group;
  const int keys = xattn_keys(a, b), nb = (keys + kTcOther - 1) / kTcOther, per = (nb + cl - 1) / cl;
  const int j_begin = min(nb, rank * per), j_end = min(nb, j_begin + per);
  const T* qb = static_cast<const T*>(a.q) + b * a.qs[0] + h * a.qs[2];
  const T* kb = static_cast<const T*>(a.k) + b * a.ks[0] + n * a.ks[2];
  const T* vb = static_cast<const T*>(a.v) + b * a.vs[0] + n * a.vs[2];
  const uint8_t* mask = a.key_mask == nullptr ? nullptr : a.key_mask + static_cast<int64_t>(b) * a.Tk;
  auto key_ok = [&](int j) { return j < keys && (mask == nullptr || __ldg(mask + j) != 0); };
  auto request = [&](int j, int buf) {
    if (j < j_end) {
      const uint32_t y = ring + buf * kTcStage;
      const int k0 = j * kTcOther;
      tc_fetch<T, kTcOther>(y, a.d, kb, [&](int i) { return key_ok(k0 + i) ? kb + (k0 + i) * a.ks[1] : nullptr; });
      tc_fetch<T, kTcOther>(y + kTcOther * 128, a.d, vb, [&](int i) { return key_ok(k0 + i) ? vb + (k0 + i) * a.vs[1] : nullptr; });
      if (tid < kTcOther) s_bias[buf][tid] = key_ok(k0 + tid) ? 0.f : -INFINITY;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  tc_fetch<T, kTcOwn>(x1, a.d, qb, [&](int i) { return own0 + i < a.Tq ? qb + (own0 + i) * a.qs[1] : nullptr; });
  request(j_begin, 0);

  float ref = kTcNone;
  float2 l2 = make_float2(0.f, 0.f);
  const float2 c2 = make_float2(a.c, a.c);
  bool ok = true;
  int it = 0;
  for (int j = j_begin; j < j_end; ++j, ++it) {
    const int buf = it & 1;
    const uint32_t y = ring + buf * kTcStage;
    if (it > 0) ok = mbar_wait(&bars[1], (it - 1) & 1);      // the sums of the block before: its buffer and P are free
    request(j + 1, buf ^ 1);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    fence_proxy_async_smem();
    tc_fence_before();
    ok = __syncthreads_and(ok);
    if (!ok) break;
    if (tid == 0) {
      tc_fence_after();
      tc_scores<T>(B.tmem + tS, x1, y);
      umma_commit(&bars[0]);
    }
    ok = __all_sync(0xffffffffu, mbar_wait(&bars[0], it & 1));
    tc_fence_after();
    if (ok) {
      float2 s[32];
      tc_read64(B.t_lane + tS, s);
      const bool plain = mask == nullptr && (j + 1) * kTcOther <= keys;
      float top = ref;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        float2 bias = make_float2(0.f, 0.f);
        if (!plain) bias = *reinterpret_cast<const float2*>(&s_bias[buf][2 * i]);
        s[i] = fma2(s[i], c2, bias);
        top = fmaxf(top, fmaxf(s[i].x, s[i].y));
      }
      if (__any_sync(0xffffffffu, top > ref + kTcSlack)) {
        const float f = ex2f(ref - top);
        ref = top;
        l2 = mul2(l2, make_float2(f, f));
        if (it > 0) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t o[16];
            tmem_ld_32x32b_x16(B.t_lane + tO + 16 * q, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_st_32x32b_x16(B.t_lane + tO + 16 * q, o);
          }
        }
      }
      const float2 m2 = make_float2(-ref, -ref);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint32_t out[32];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float2 p = add2(s[16 * q + i], m2);
          p.x = ex2f(p.x), p.y = ex2f(p.y);
          l2 = add2(l2, p);
          tc_split<T>(p, out, i);
        }
        tmem_st_32x32b_x32(B.t_lane + tS + 32 * q, out);
      }
      tmem_st_wait();
    }
    tc_fence_before();
    ok = __syncthreads_and(ok);
    if (!ok) break;
    if (tid == 0) {
      tc_fence_after();
      tc_sums<T>(B.tmem + tO, B.tmem + tS, y + kTcOther * 128, it > 0);
      umma_commit(&bars[1]);
    }
  }
  if (ok && it > 0) ok = mbar_wait(&bars[1], (it - 1) & 1);
  tc_fence_after();
  __syncwarp();
  float2 o[32];
  if (it > 0) {
    tc_read64(B.t_lane + tO, o);
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) o[i] = make_float2(0.f, 0.f);
  }
  B.close(128);
  const float l = l2.x + l2.y;
  const int64_t stat0 = (static_cast<int64_t>(b) * a.heads + h) * a.Tq;
  auto to_row = [&](int r) { return static_cast<T*>(a.out) + b * a.os[0] + r * a.os[1] + h * a.os[2]; };
  auto to_row32 = [&](int r) { return a.out_f32 + ((static_cast<int64_t>(b) * a.Tq + r) * a.heads + h) * a.d; };
  if (cl == 1) {
    const int r = own0 + tid;
    if (r < a.Tq) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      tc_store_row<T>(to_row(r), a.d, o, inv);
      if (a.out_f32 != nullptr) {
#pragma unroll
        for (int c = 0; c < 16; ++c)
          if (c * 4 < a.d)
            *reinterpret_cast<float4*>(to_row32(r) + c * 4) =
                make_float4(o[2 * c].x * inv, o[2 * c].y * inv, o[2 * c + 1].x * inv, o[2 * c + 1].y * inv);
      }
      if (a.lse != nullptr) a.lse[stat0 + r] = l == 0.f ? INFINITY : ref + log2f(l);
    }
  } else {
    s_ref[tid] = ref, s_l[tid] = l;
    tc_put64(ring, tid, o, 1.f);
    cluster_sync_all();
    // 16 threads join a row: its blocks' sums at their highest reference
    for (int i = tid / 16; i * cl + rank < kTcOwn; i += kTcThreads / 16) {
      const int row = i * cl + rank, c = tid % 16, r = own0 + row;
      float m = kTcNone, den = 0.f;
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int z = 0; z < cl; ++z) m = fmaxf(m, ld_dsmem(mapa_shared(smem_u32(&s_ref[row]), z)));
      for (int z = 0; z < cl; ++z) {
        const float f = ex2f(ld_dsmem(mapa_shared(smem_u32(&s_ref[row]), z)) - m);
        den = fmaf(ld_dsmem(mapa_shared(smem_u32(&s_l[row]), z)), f, den);
        const float4 v = ld_dsmem4(mapa_shared(tc_join_chunk(ring, row, c), z));
        y = make_float4(fmaf(v.x, f, y.x), fmaf(v.y, f, y.y), fmaf(v.z, f, y.z), fmaf(v.w, f, y.w));
      }
      if (r >= a.Tq) continue;
      const float inv = den == 0.f ? 0.f : 1.f / den;
      y = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
      if (c * 4 < a.d) {
        *reinterpret_cast<uint2*>(to_row(r) + c * 4) = make_uint2(tc_pack<T>(y.x, y.y), tc_pack<T>(y.z, y.w));
        if (a.out_f32 != nullptr) *reinterpret_cast<float4*>(to_row32(r) + c * 4) = y;
      }
      if (a.lse != nullptr && c == 0) a.lse[stat0 + r] = den == 0.f ? INFINITY : m + log2f(den);
    }
    cluster_sync_all();
  }
}

// OWN_ROWS: a tile of queries, x = q, dout, over keys, y = k, v: dq += dS k, and D is left for the keys' kernel.
// Else a tile of keys, x = k, v, over the queries of its heads, y = q, dout: dk += dS q, dv += P dout.
template <bool OWN_ROWS>
__global__ void __launch_bounds__(kTcThreads, 2) xattn_tc_bwd_kernel(const XAttn a) {
  using T = __nv_bfloat16;
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t bars[2];
  __shared__ uint32_t holder;
  __shared__ __align__(16) float s_a[2][kTcOther], s_b[2][kTcOther];   // of the other side: bias; or -lse and -D
  TcBlock B;
  B.open(raw, bars, &holder, 256);
  const uint32_t x1 = B.sm, x2 = B.sm + kTcTile, ring = B.sm + 2 * kTcTile, tS = 0, tD = 64, tA1 = 128, tA2 = 192;
  const int tid = threadIdx.x;
  const int cl = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
  const int own0 = static_cast<int>(blockIdx.x) / cl * kTcOwn, b = blockIdx.z;
  const int h0 = OWN_ROWS ? blockIdx.y : blockIdx.y * a.group, n = OWN_ROWS ? h0 / a.group : blockIdx.y;
  const int keys = xattn_keys(a, b);
  const int qblocks = (a.Tq + kTcOther - 1) / kTcOther;
  const int nb = OWN_ROWS ? (keys + kTcOther - 1) / kTcOther : own0 < keys ? a.group * qblocks : 0, per = (nb + cl - 1) / cl;
  const int j_begin = min(nb, rank * per);
  const int j_end = OWN_ROWS && a.dq == nullptr ? j_begin : min(nb, j_begin + per);   // only D was wanted
  const T* qb = static_cast<const T*>(a.q) + b * a.qs[0];
  const T* ob = static_cast<const T*>(a.dout) + b * a.os[0];
  const T* kb = static_cast<const T*>(a.k) + b * a.ks[0] + n * a.ks[2];
  const T* vb = static_cast<const T*>(a.v) + b * a.vs[0] + n * a.vs[2];
  const uint8_t* mask = a.key_mask == nullptr ? nullptr : a.key_mask + static_cast<int64_t>(b) * a.Tk;
  auto key_ok = [&](int j) { return j < keys && (mask == nullptr || __ldg(mask + j) != 0); };
  auto stat = [&](int h) { return (static_cast<int64_t>(b) * a.heads + h) * a.Tq; };
  auto request = [&](int j, int buf) {
    if (j < j_end) {
      const uint32_t y = ring + buf * kTcStage, y2 = y + kTcOther * 128;
      if constexpr (OWN_ROWS) {
        const int k0 = j * kTcOther;
        tc_fetch<T, kTcOther>(y, a.d, kb, [&](int i) { return key_ok(k0 + i) ? kb + (k0 + i) * a.ks[1] : nullptr; });
        tc_fetch<T, kTcOther>(y2, a.d, vb, [&](int i) { return key_ok(k0 + i) ? vb + (k0 + i) * a.vs[1] : nullptr; });
        if (tid < kTcOther) s_a[buf][tid] = key_ok(k0 + tid) ? 0.f : -INFINITY;
      } else {
        const int h = h0 + j / qblocks, t0 = j % qblocks * kTcOther;
        tc_fetch<T, kTcOther>(y, a.d, qb, [&](int i) { return t0 + i < a.Tq ? qb + (t0 + i) * a.qs[1] + h * a.qs[2] : nullptr; });
        tc_fetch<T, kTcOther>(y2, a.d, ob, [&](int i) { return t0 + i < a.Tq ? ob + (t0 + i) * a.os[1] + h * a.os[2] : nullptr; });
        const int t = t0 + tid % kTcOther;
        float* to = tid < kTcOther ? s_a[buf] : s_b[buf];
        const float* from = tid < kTcOther ? a.lse : a.delta;
        to[tid % kTcOther] = t < a.Tq ? -__ldg(from + stat(h) + t) : (tid < kTcOther ? -INFINITY : 0.f);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  float own_s, own_d = 0.f;                  // -lse and -D of the thread's query; bias of its key
  const int mine = own0 + tid;
  if constexpr (OWN_ROWS) {
    const T *q = qb + h0 * a.qs[2], *o = ob + h0 * a.os[2];
    tc_fetch<T, kTcOwn>(x1, a.d, q, [&](int i) { return own0 + i < a.Tq ? q + (own0 + i) * a.qs[1] : nullptr; });
    tc_fetch<T, kTcOwn>(x2, a.d, o, [&](int i) { return own0 + i < a.Tq ? o + (own0 + i) * a.os[1] : nullptr; });
    request(j_begin, 0);
    own_s = -INFINITY;
    if (mine < a.Tq) {
      own_s = -__ldg(a.lse + stat(h0) + mine);
      const float* o32 = a.out_f32 + ((static_cast<int64_t>(b) * a.Tq + mine) * a.heads + h0) * a.d;
      for (int c = 0; c < a.d; c += 8) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(o + mine * a.os[1] + c));
        const float4 f0 = __ldg(reinterpret_cast<const float4*>(o32 + c)), f1 = __ldg(reinterpret_cast<const float4*>(o32 + c + 4));
        const float2 g0 = tc_unpack<T>(u.x), g1 = tc_unpack<T>(u.y), g2 = tc_unpack<T>(u.z), g3 = tc_unpack<T>(u.w);
        own_d = fmaf(-f0.x, g0.x, fmaf(-f0.y, g0.y, fmaf(-f0.z, g1.x, fmaf(-f0.w, g1.y, own_d))));
        own_d = fmaf(-f1.x, g2.x, fmaf(-f1.y, g2.y, fmaf(-f1.z, g3.x, fmaf(-f1.w, g3.y, own_d))));
      }
      if (rank == 0) a.delta[stat(h0) + mine] = -own_d;
    }
  } else {
    tc_fetch<T, kTcOwn>(x1, a.d, kb, [&](int i) { return key_ok(own0 + i) ? kb + (own0 + i) * a.ks[1] : nullptr; });
    tc_fetch<T, kTcOwn>(x2, a.d, vb, [&](int i) { return key_ok(own0 + i) ? vb + (own0 + i) * a.vs[1] : nullptr; });
    request(j_begin, 0);
    own_s = key_ok(mine) ? 0.f : -INFINITY;
  }

  const float2 c2 = make_float2(a.c, a.c), os2 = make_float2(own_s, own_s), od2 = make_float2(own_d, own_d);
  bool ok = true;
  int it = 0;
  for (int j = j_begin; j < j_end; ++j, ++it) {
    const int buf = it & 1;
    const uint32_t y = ring + buf * kTcStage, y2 = y + kTcOther * 128;
    if (it > 0) ok = mbar_wait(&bars[1], (it - 1) & 1);
    request(j + 1, buf ^ 1);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    fence_proxy_async_smem();
    tc_fence_before();
    ok = __syncthreads_and(ok);
    if (!ok) break;
    if (tid == 0) {
      tc_fence_after();
      tc_scores<T>(B.tmem + tS, x1, y);
      tc_scores<T>(B.tmem + tD, x2, y2);
      umma_commit(&bars[0]);
    }
    ok = __all_sync(0xffffffffu, mbar_wait(&bars[0], it & 1));
    tc_fence_after();
    if (ok) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint32_t rs[32], rd[32], ps[32], pd[32];
        tmem_ld_32x32b_x32(B.t_lane + tS + 32 * q, rs);
        tmem_ld_32x32b_x32(B.t_lane + tD + 32 * q, rd);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float2 sa = *reinterpret_cast<const float2*>(&s_a[buf][32 * q + 2 * i]);
          float2 p = fma2(make_float2(__uint_as_float(rs[2 * i]), __uint_as_float(rs[2 * i + 1])), c2, OWN_ROWS ? sa : os2);
          p = add2(p, OWN_ROWS ? os2 : sa);
          p.x = ex2f(p.x), p.y = ex2f(p.y);
          const float2 dd = OWN_ROWS ? od2 : *reinterpret_cast<const float2*>(&s_b[buf][32 * q + 2 * i]);
          const float2 ds = mul2(p, add2(make_float2(__uint_as_float(rd[2 * i]), __uint_as_float(rd[2 * i + 1])), dd));
          tc_split<T>(ds, pd, i);
          if constexpr (!OWN_ROWS) tc_split<T>(p, ps, i);
        }
        tmem_st_32x32b_x32(B.t_lane + tD + 32 * q, pd);
        if constexpr (!OWN_ROWS) tmem_st_32x32b_x32(B.t_lane + tS + 32 * q, ps);
      }
      tmem_st_wait();
    }
    tc_fence_before();
    ok = __syncthreads_and(ok);
    if (!ok) break;
    if (tid == 0) {
      tc_fence_after();
      tc_sums<T>(B.tmem + tA1, B.tmem + tD, y, it > 0);
      if constexpr (!OWN_ROWS) tc_sums<T>(B.tmem + tA2, B.tmem + tS, y2, it > 0);
      umma_commit(&bars[1]);
    }
  }
  if (ok && it > 0) ok = mbar_wait(&bars[1], (it - 1) & 1);
  tc_fence_after();
  __syncwarp();
  auto to_row = [&](void* to, int r) {
    return static_cast<T*>(to) + (OWN_ROWS ? (static_cast<int64_t>(b) * a.Tq + r) * a.heads + h0
                                           : (static_cast<int64_t>(b) * a.Tk + r) * a.kv_heads + n) * a.d;
  };
  const int rows = OWN_ROWS ? a.Tq : a.Tk;
  if (cl > 1) {                              // the operands' memory takes the sums: 32 KB of ring, 32 KB of x1, x2
    cp_async_wait_all();
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < (OWN_ROWS ? 1 : 2); ++k) {
    float2 v[32];
    if (it > 0) {
      tc_read64(B.t_lane + (k == 0 ? tA1 : tA2), v);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = make_float2(0.f, 0.f);
    }
    const float f = k == 0 ? a.scale : 1.f;
    void* to = OWN_ROWS ? a.dq : k == 0 ? a.dk : a.dv;
    if (cl > 1) {
      tc_put64(k == 0 ? ring : x1, tid, v, f);
    } else if (mine < rows && to != nullptr) {
      tc_store_row<T>(to_row(to, mine), a.d, v, f);
    }
  }
  B.close(256);
  if (cl == 1) return;
  cluster_sync_all();
#pragma unroll
  for (int k = 0; k < (OWN_ROWS ? 1 : 2); ++k) {
    void* to = OWN_ROWS ? a.dq : k == 0 ? a.dk : a.dv;
    const uint32_t tile = k == 0 ? ring : x1;
    for (int i = tid / 16; i * cl + rank < kTcOwn; i += kTcThreads / 16) {
      const int row = i * cl + rank, c = tid % 16, r = own0 + row;
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int z = 0; z < cl; ++z) {
        const float4 u = ld_dsmem4(mapa_shared(tc_join_chunk(tile, row, c), z));
        y = make_float4(y.x + u.x, y.y + u.y, y.z + u.z, y.w + u.w);
      }
      if (r < rows && c * 4 < a.d && to != nullptr)
        *reinterpret_cast<uint2*>(to_row(to, r) + c * 4) = make_uint2(tc_pack<T>(y.x, y.y), tc_pack<T>(y.z, y.w));
    }
  }
  cluster_sync_all();
}

// Blocks per cluster: the other side is split until the device's slots (per_sm blocks each) are taken, with two steps
// left to each block.
static int xattn_tc_cluster(int64_t blocks, int per_sm, int steps) {
  const int64_t c = 148 * per_sm / blocks;
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({c, 8, steps / 2})));
}
template <class K>
static int xattn_tc_launch(K kernel, PerDeviceOnce& once, dim3 grid, int smem, int cl, cudaStream_t stream, const XAttn& a) {
  const int st = allow_smem(once, kernel, smem);
  if (st != SSAM_OK) return st;
  cudaLaunchConfig_t cfg = {};
  grid.x *= cl;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kTcThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cl;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return status_from_cuda(cudaLaunchKernelEx(&cfg, kernel, a));
}

template <class T>
static int xattn_tc_fwd_t(const XAttn& a, cudaStream_t stream) {
  static PerDeviceOnce once;
  const int tiles = (a.Tq + kTcOwn - 1) / kTcOwn;
  const int cl = xattn_tc_cluster(static_cast<int64_t>(a.B) * a.heads * tiles, 4, (a.Tk + kTcOther - 1) / kTcOther);
  return xattn_tc_launch(xattn_tc_fwd_kernel<T>, once, dim3(tiles, a.heads, a.B), kTcTile + 2 * kTcStage + 1024, cl, stream, a);
}
int xattn_tc_fwd(const XAttn& a, int dtype, cudaStream_t stream) {
  return dtype == 0 ? xattn_tc_fwd_t<__half>(a, stream) : xattn_tc_fwd_t<__nv_bfloat16>(a, stream);
}
int xattn_tc_bwd(const XAttn& a, cudaStream_t stream) {
  static PerDeviceOnce by_rows, by_keys;
  constexpr int smem = 2 * kTcTile + 2 * kTcStage + 1024;
  int tiles = (a.Tq + kTcOwn - 1) / kTcOwn;
  int cl = xattn_tc_cluster(static_cast<int64_t>(a.B) * a.heads * tiles, 2, (a.Tk + kTcOther - 1) / kTcOther);
  const int st = xattn_tc_launch(xattn_tc_bwd_kernel<true>, by_rows, dim3(tiles, a.heads, a.B), smem, cl, stream, a);
  if (st != SSAM_OK || a.dk == nullptr) return st;
  tiles = (a.Tk + kTcOwn - 1) / kTcOwn;
  cl = xattn_tc_cluster(static_cast<int64_t>(a.B) * a.kv_heads * tiles, 2, a.group * ((a.Tq + kTcOther - 1) / kTcOther));
  return xattn_tc_launch(xattn_tc_bwd_kernel<false>, by_keys, dim3(tiles, a.kv_heads, a.B), smem, cl, stream, a);
}

}  // namespace ssam
