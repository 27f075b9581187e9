// Cross attention of two long sides on the 5th-generation tensor cores (formulas and conventions in
// cross_attention.cuh): fp16 and bf16, heads of up to 128 channels, zero-padded to NP panels of 64.
//
// A block owns a tile of 128 entries of one side (an entry is a TMEM lane and a thread; two threads in the backward
// pass) and walks the other side 64 entries at a time:
//   S = X1 Y1^T (and dP = X2 Y2^T)      tcgen05.mma, both operands in shared memory, K-major, 128-byte swizzle
//   P (and dS) from S by its thread     tcgen05.ld, exponentials, tcgen05.st over the columns of S (and dP)
//   sums += P Y2, dS Y1                 tcgen05.mma with the first operand in TMEM; the same shared-memory tile now
//                                       MN-major (its rows are the k axis)
// P and dS enter as two half terms: of every 16 fp32 columns, the first 8 take the values, the others the remainders.
// These products run in bf16 for fp16 inputs too (fp16 ends at 2^-24, and small weights count where the large ones meet
// zeros; the sums in TMEM have no room for the scheme of cross_attention_mma.cuh): the other side's tile becomes two
// bf16 tiles once the scores are there, its values in place and its remainders over a tile that is free by then (V's over
// K, K's over V) or, in the keys' kernel, which needs both its tiles, behind the ring. Products with P take all four
// pairs of terms: two terms of P are within 2^-17 of it, and the pair of the remainders is up to 2^-16 of a product.
// Those with dS leave that pair out, next to the roundings of dP - D.
// The chain load -> mma -> softmax -> mma of a block is serial; 4 (forward: 128 TMEM columns) or 2 (backward: 256)
// blocks per SM run each other's gaps. Tiles come by cp.async rather than TMA: rows of masked keys and channels past
// d are zero-filled on the way, and any row stride will do. Where tiles leave the device empty, the other side is
// split over a cluster and joined through distributed shared memory in rank order.
// Every wait is bounded; a block whose wait ran out raises SSAM_ERR_TIMEOUT and leaves.
//
// Bound by that chain: 1369 x 4096, 2 x 4 heads of 64, bf16, takes 41 us forward (280 TFLOP/s) and 149 with the
// gradients (fp16, with its further products, 48 and 180), at 20 to 28 % of the tensor pipe, 18 to 29 % of the
// exponentials' and 41 to 47 % of the issue slots. mma.sync on registers took 60 and 339. Two threads per row in the forward kernel (64 registers) were slower: 161.
#include <cuda_fp16.h>

#include "common.cuh"
#include "cross_attention.cuh"
#include "host_util.h"

namespace ssam {

constexpr int kTcOwn = 128, kTcOther = 64, kTcThreads = 128;
constexpr int kTcTile = kTcOwn * 128, kTcHalf = kTcOther * 128;   // bytes of a panel of the own and of the other side

// 16-byte chunk c (8 channels) of row r of a 128-byte-swizzled tile
__device__ __forceinline__ uint32_t tc_chunk(uint32_t tile, int r, int c) { return tile + r * 128 + ((c ^ (r & 7)) << 4); }

// Starts the copies of ROWS rows (row(i): address, nullptr: zeros) into a tile by THREADS threads.
template <class T, int NP, int ROWS, int THREADS, class R>
__device__ __forceinline__ void tc_fetch(uint32_t tile, int d, const T* valid, R row) {
  const int c = threadIdx.x % (8 * NP);
#pragma unroll
  for (int i0 = 0; i0 < ROWS; i0 += THREADS / (8 * NP)) {
    const int i = i0 + threadIdx.x / (8 * NP);
    const T* p = row(i);
    const bool there = p != nullptr && c * 8 < d;
    cp_async16(tc_chunk(tile + c / 8 * (ROWS * 128), i, c % 8), there ? p + c * 8 : valid, there ? 16u : 0u);
  }
}
template <class T>
constexpr uint32_t tc_idesc(uint32_t b_mn) {
  const uint32_t f = sizeof(T) == 2 && std::is_same<T, __half>::value ? 0u : 1u;
  return (1u << 4) | (f << 7) | (f << 10) | (b_mn << 16) | ((64u >> 3) << 17) | ((128u >> 4) << 24);
}
// D[128 x 64] = A[128 x channels] B[64 entries x channels]^T
template <class T, int NP>
__device__ __forceinline__ void tc_scores(uint32_t d_tmem, uint32_t a, uint32_t b) {
#pragma unroll
  for (int k = 0; k < 4 * NP; ++k)
    umma_f16_ss(d_tmem, make_smem_desc(a + k / 4 * kTcTile + k % 4 * 32, 16, 1024, kSw128),
                make_smem_desc(b + k / 4 * kTcHalf + k % 4 * 32, 16, 1024, kSw128), tc_idesc<T>(0), k > 0);
}
// D[128 x channels] (+)= P[128 x 64 entries] B[64 entries x channels] in bf16, P in TMEM as [8 values | 8 remainders] four
// times; TERMS: B's remainders are at b_lo, and their product with P's values (1), and remainders too (2), is added
template <int NP, int TERMS>
__device__ __forceinline__ void tc_sums(uint32_t d_tmem, uint32_t p_tmem, uint32_t b, uint32_t b_lo, bool accumulate) {
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const uint64_t desc = make_smem_desc(b + p * kTcHalf + k * 2048, 16, 1024, kSw128);
      umma_f16_ts(d_tmem + 64 * p, p_tmem + k * 16, desc, tc_idesc<__nv_bfloat16>(1), accumulate || k > 0);
      umma_f16_ts(d_tmem + 64 * p, p_tmem + k * 16 + 8, desc, tc_idesc<__nv_bfloat16>(1), 1u);
      if constexpr (TERMS > 0) {
        const uint64_t lo = make_smem_desc(b_lo + p * kTcHalf + k * 2048, 16, 1024, kSw128);
        umma_f16_ts(d_tmem + 64 * p, p_tmem + k * 16, lo, tc_idesc<__nv_bfloat16>(1), 1u);
        if constexpr (TERMS > 1) umma_f16_ts(d_tmem + 64 * p, p_tmem + k * 16 + 8, lo, tc_idesc<__nv_bfloat16>(1), 1u);
      }
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
// value pair i of 16 columns -> out[i] (values), out[8 + i] (remainders)
__device__ __forceinline__ void tc_split(float2 p, uint32_t (&out)[16], int i) {
  out[i] = pack_bf16x2(p.x, p.y);
  const float2 h = tc_unpack<__nv_bfloat16>(out[i]), r = add2(p, make_float2(-h.x, -h.y));
  out[8 + i] = pack_bf16x2(r.x, r.y);
}
// A landed fp16 tile of the other side as bf16 terms: the values in place, the remainders at `lo`, laid out alike.
template <int NP, int THREADS>
__device__ __forceinline__ void tc_terms(uint32_t tile, uint32_t lo) {
  static_assert(kTcHalf % (THREADS * 16) == 0, "every thread has the same number of chunks");
#pragma unroll
  for (int i = 0; i < NP * kTcHalf / (THREADS * 16); ++i) {
    const uint32_t o = (i * THREADS + threadIdx.x) * 16;
    uint32_t h[4], l[4];
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(tile + o) : "memory");
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = tc_unpack<__half>(h[e]);
      h[e] = pack_bf16x2(f.x, f.y);
      const float2 v = tc_unpack<__nv_bfloat16>(h[e]), r = add2(f, make_float2(-v.x, -v.y));
      l[e] = pack_bf16x2(r.x, r.y);
    }
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(tile + o), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(lo + o), "r"(l[0]), "r"(l[1]), "r"(l[2]), "r"(l[3]) : "memory");
  }
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
// Puts 4 N of row r's sums, times f, into the join's tile from chunk c0 on.
template <int N>
__device__ __forceinline__ void tc_put(uint32_t tile, int r, int c0, const float2 (&v)[2 * N], float f) {
#pragma unroll
  for (int c = 0; c < N; ++c)
    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(tc_join_chunk(tile, r, c0 + c)), "f"(v[2 * c].x * f),
                 "f"(v[2 * c].y * f), "f"(v[2 * c + 1].x * f), "f"(v[2 * c + 1].y * f)
                 : "memory");
}
// Stores 8 N channels of a row, as far as d goes.
template <class T, int N>
__device__ __forceinline__ void tc_store_row(T* to, int d, const float2 (&v)[4 * N], float f) {
#pragma unroll
  for (int c = 0; c < N; ++c)
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
    t_lane = tmem + (threadIdx.x / 32 % 4 * 32u << 16);
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
// Every thread's copies (into shared memory) and TMEM stores are there for the tensor core.
__device__ __forceinline__ bool tc_landed(bool ok) {
  cp_async_wait_all();
  fence_proxy_async_smem();
  tc_fence_before();
  return __syncthreads_and(ok);
}
constexpr float kTcNone = -3.402823466e38f, kTcSlack = 8.f;   // no finite logit is below the first

// Folded row r of key head n is token r % Tq of query head n group + r / Tq.
struct TcRow {
  int64_t t, h;
};
__device__ __forceinline__ TcRow tc_row(const XAttn& a, int n, int r) {
  const int g = a.group == 1 ? 0 : r / a.Tq;
  return {r - g * a.Tq, n * a.group + g};
}

template <class T, int NP>
__global__ void __launch_bounds__(kTcThreads, 4 / NP) xattn_tc_fwd_kernel(const XAttn args) {
  const XAttn a = follow(args, true);
  constexpr int kTile = NP * kTcTile, kHalfStage = NP * kTcHalf, kStage = 2 * kHalfStage, kCols = 128 * NP;
  constexpr bool kTerms = std::is_same<T, __half>::value;
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t bars[2];
  __shared__ uint32_t holder;
  __shared__ __align__(16) float s_bias[2][kTcOther];
  __shared__ float s_ref[kTcOwn], s_l[kTcOwn];
  TcBlock B;
  B.open(raw, bars, &holder, kCols);
  const uint32_t x1 = B.sm, ring = B.sm + kTile, tS = 0, tO = 64;
  const int tid = threadIdx.x;
  const int cl = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
  const int own0 = static_cast<int>(blockIdx.x) / cl * kTcOwn, n = blockIdx.y, b = blockIdx.z, rows = a.group * a.Tq;
  const int keys = xattn_keys(a, b), nb = (keys + kTcOther - 1) / kTcOther, per = (nb + cl - 1) / cl;
  const int j_begin = min(nb, rank * per), j_end = min(nb, j_begin + per);
  const T* qb = static_cast<const T*>(a.q) + b * a.qs[0];
  const T* kb = static_cast<const T*>(a.k) + b * a.ks[0] + n * a.ks[2];
  const T* vb = static_cast<const T*>(a.v) + b * a.vs[0] + n * a.vs[2];
  const uint8_t* mask = a.key_mask == nullptr ? nullptr : a.key_mask + static_cast<int64_t>(b) * a.Tk;
  auto key_ok = [&](int j) { return j < keys && (mask == nullptr || __ldg(mask + j) != 0); };
  bool some = false;                         // one of the keys that this thread looked at is there
  auto request = [&](int j, int buf) {
    if (j < j_end) {
      const uint32_t y = ring + buf * kStage;
      const int k0 = j * kTcOther;
      tc_fetch<T, NP, kTcOther, kTcThreads>(y, a.d, kb, [&](int i) { return key_ok(k0 + i) ? kb + (k0 + i) * a.ks[1] : nullptr; });
      tc_fetch<T, NP, kTcOther, kTcThreads>(y + kHalfStage, a.d, vb,
                                            [&](int i) { return key_ok(k0 + i) ? vb + (k0 + i) * a.vs[1] : nullptr; });
      if (tid < kTcOther) {
        const bool there = key_ok(k0 + tid);
        s_bias[buf][tid] = there ? 0.f : -INFINITY;
        some |= there;
      }
    }
  };
  tc_fetch<T, NP, kTcOwn, kTcThreads>(x1, a.d, qb, [&](int i) -> const T* {
    if (own0 + i >= rows) return nullptr;
    const TcRow r = tc_row(a, n, own0 + i);
    return qb + r.t * a.qs[1] + r.h * a.qs[2];
  });
  request(j_begin, 0);

  float ref = kTcNone;
  float2 l2 = make_float2(0.f, 0.f);
  const float2 c2 = make_float2(a.c, a.c);
  bool ok = tc_landed(true);
  int it = 0;
  for (int j = j_begin; j < j_end; ++j, ++it) {
    const int buf = it & 1;
    const uint32_t y = ring + buf * kStage;
    if (it > 0) ok = mbar_wait(&bars[1], (it - 1) & 1);      // the sums of the step before: its buffer and P are free
    if (tid == 0 && ok) {
      tc_fence_after();
      tc_scores<T, NP>(B.tmem + tS, x1, y);
      umma_commit(&bars[0]);
    }
    request(j + 1, buf ^ 1);
    ok = __all_sync(0xffffffffu, ok && mbar_wait(&bars[0], it & 1));
    tc_fence_after();
    if (ok) {
      if constexpr (kTerms) tc_terms<NP, kTcThreads>(y + kHalfStage, y);
      float2 s[32];
      tc_read64(B.t_lane + tS, s);
      const bool plain = mask == nullptr && (j + 1) * kTcOther <= keys;
      if (plain) {
#pragma unroll
        for (int i = 0; i < 32; ++i) s[i] = mul2(s[i], c2);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) s[i] = fma2(s[i], c2, *reinterpret_cast<const float2*>(&s_bias[buf][2 * i]));
      }
      float top = ref;
#pragma unroll
      for (int i = 0; i < 32; ++i) top = fmaxf(top, fmaxf(s[i].x, s[i].y));
      if (__any_sync(0xffffffffu, top > ref + kTcSlack)) {
        const float f = ex2f(ref - top);
        ref = top;
        l2 = mul2(l2, make_float2(f, f));
        if (it > 0) {
#pragma unroll
          for (int q = 0; q < 4 * NP; ++q) {
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
      for (int q = 0; q < 4; ++q) {
        uint32_t out[16];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float2 p = add2(s[8 * q + i], m2);
          p.x = ex2f(p.x), p.y = ex2f(p.y);
          l2 = add2(l2, p);
          tc_split(p, out, i);
        }
        tmem_st_32x32b_x16(B.t_lane + tS + 16 * q, out);
      }
      tmem_st_wait();
    }
    ok = tc_landed(ok);
    if (!ok) break;
    if (tid == 0) {
      tc_fence_after();
      tc_sums<NP, kTerms ? 2 : 0>(B.tmem + tO, B.tmem + tS, y + kHalfStage, y, it > 0);
      umma_commit(&bars[1]);
    }
  }
  if (ok && it > 0) ok = mbar_wait(&bars[1], (it - 1) & 1);
  tc_fence_after();
  __syncwarp();
  // where every key that was walked is masked, a query that is not finite leaves NaN, which is nothing's
  const bool any = it > 0 && (mask == nullptr || __syncthreads_or(some));
  if (!any) ref = kTcNone, l2 = make_float2(0.f, 0.f);
  const float l = l2.x + l2.y;
  const float inv = cl > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
  const int64_t stat0 = (static_cast<int64_t>(b) * a.heads + n * a.group) * a.Tq;
  auto to_row = [&](const TcRow& r) { return static_cast<T*>(a.out) + b * a.os[0] + r.t * a.os[1] + r.h * a.os[2]; };
  auto to_row32 = [&](const TcRow& r) { return a.out_f32 + ((static_cast<int64_t>(b) * a.Tq + r.t) * a.heads + r.h) * a.d; };
  if (cl > 1) cp_async_wait_all(), __syncthreads();    // the ring takes the sums
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    float2 o[32];
    if (any) {
      tc_read64(B.t_lane + tO + 64 * p, o);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] = make_float2(0.f, 0.f);
    }
    const int r = own0 + tid, d = a.d - 64 * p;
    if (cl > 1) {
      tc_put<16>(ring + p * 2 * kTcTile, tid, 0, o, 1.f);
    } else if (r < rows) {
      const TcRow at = tc_row(a, n, r);
      tc_store_row<T, 8>(to_row(at) + 64 * p, d, o, inv);
      if (a.out_f32 != nullptr) {
#pragma unroll
        for (int c = 0; c < 16; ++c)
          if (c * 4 < d)
            *reinterpret_cast<float4*>(to_row32(at) + 64 * p + c * 4) =
                make_float4(o[2 * c].x * inv, o[2 * c].y * inv, o[2 * c + 1].x * inv, o[2 * c + 1].y * inv);
      }
    }
  }
  B.close(kCols);
  if (cl == 1) {
    if (own0 + tid < rows && a.lse != nullptr) a.lse[stat0 + own0 + tid] = l == 0.f ? INFINITY : ref + log2f(l);
  } else {
    s_ref[tid] = ref, s_l[tid] = l;
    cluster_sync_all();
    // 16 threads join a row: its blocks' sums at their highest reference
    for (int i = tid / 16; i * cl + rank < kTcOwn; i += kTcThreads / 16) {
      const int row = i * cl + rank, c = tid % 16, r = own0 + row;
      if (r >= rows) continue;
      float m = kTcNone, den = 0.f;
      for (int z = 0; z < cl; ++z) m = fmaxf(m, ld_dsmem(mapa_shared(smem_u32(&s_ref[row]), z)));
      for (int z = 0; z < cl; ++z)
        den = fmaf(ld_dsmem(mapa_shared(smem_u32(&s_l[row]), z)), ex2f(ld_dsmem(mapa_shared(smem_u32(&s_ref[row]), z)) - m), den);
      const float inv_den = den == 0.f ? 0.f : 1.f / den;
      const TcRow at = tc_row(a, n, r);
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int z = 0; z < cl; ++z) {
          const float f = ex2f(ld_dsmem(mapa_shared(smem_u32(&s_ref[row]), z)) - m);
          const float4 v = ld_dsmem4(mapa_shared(tc_join_chunk(ring + p * 2 * kTcTile, row, c), z));
          y = make_float4(fmaf(v.x, f, y.x), fmaf(v.y, f, y.y), fmaf(v.z, f, y.z), fmaf(v.w, f, y.w));
        }
        y = make_float4(y.x * inv_den, y.y * inv_den, y.z * inv_den, y.w * inv_den);
        const int at_c = 64 * p + c * 4;
        if (at_c < a.d) {
          *reinterpret_cast<uint2*>(to_row(at) + at_c) = make_uint2(tc_pack<T>(y.x, y.y), tc_pack<T>(y.z, y.w));
          if (a.out_f32 != nullptr) *reinterpret_cast<float4*>(to_row32(at) + at_c) = y;
        }
      }
      if (a.lse != nullptr && c == 0) a.lse[stat0 + r] = den == 0.f ? INFINITY : m + log2f(den);
    }
    cluster_sync_all();
  }
}

// OWN_ROWS: a tile of queries, x = q, dout, over keys, y = k, v: dq += dS k, and D is left for the keys' kernel.
// Else a tile of keys, x = k, v, over the queries of its heads, y = q, dout: dk += dS q, dv += P dout.
// Two threads share an entry, 32 columns each (warps w and w + 4 reach the same TMEM lanes).
constexpr int kTcBwdThreads = 256;

template <class T, int NP, bool OWN_ROWS>
__global__ void __launch_bounds__(kTcBwdThreads, 2 / NP) xattn_tc_bwd_kernel(const XAttn args) {
  const XAttn a = follow(args, true);
  constexpr bool kTerms = std::is_same<T, __half>::value;
  constexpr int kTile = NP * kTcTile, kHalfStage = NP * kTcHalf, kStage = 2 * kHalfStage;
  constexpr int kCols = NP == 1 || OWN_ROWS ? 256 : 512;
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t bars[2];
  __shared__ uint32_t holder;
  __shared__ __align__(16) float s_a[2][kTcOther], s_b[2][kTcOther];   // of the other side: bias; or -lse and -D
  __shared__ float s_d[OWN_ROWS ? kTcOwn : 1];
  TcBlock B;
  B.open(raw, bars, &holder, kCols);
  const uint32_t x1 = B.sm, x2 = B.sm + kTile, ring = B.sm + 2 * kTile, tS = 0, tD = 64, tA1 = 128, tA2 = 128 + 64 * NP;
  const int tid = threadIdx.x, lane_id = tid % kTcOwn, half = tid / kTcOwn;
  const int cl = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
  const int own0 = static_cast<int>(blockIdx.x) / cl * kTcOwn, n = blockIdx.y, b = blockIdx.z;
  const int rows = a.group * a.Tq, keys = xattn_keys(a, b);
  const int nb = ((OWN_ROWS ? keys : own0 < keys ? rows : 0) + kTcOther - 1) / kTcOther, per = (nb + cl - 1) / cl;
  const int j_begin = min(nb, rank * per);
  const int j_end = OWN_ROWS && a.dq == nullptr ? j_begin : min(nb, j_begin + per);   // only D was wanted
  const T* qb = static_cast<const T*>(a.q) + b * a.qs[0];
  const T* ob = static_cast<const T*>(a.dout) + b * a.os[0];
  const T* kb = static_cast<const T*>(a.k) + b * a.ks[0] + n * a.ks[2];
  const T* vb = static_cast<const T*>(a.v) + b * a.vs[0] + n * a.vs[2];
  const uint8_t* mask = a.key_mask == nullptr ? nullptr : a.key_mask + static_cast<int64_t>(b) * a.Tk;
  const int64_t stat0 = (static_cast<int64_t>(b) * a.heads + n * a.group) * a.Tq;
  auto key_ok = [&](int j) { return j < keys && (mask == nullptr || __ldg(mask + j) != 0); };
  auto row_at = [&](const T* base, const int64_t (&s)[3], int r) -> const T* {
    if (r >= rows) return nullptr;
    const TcRow at = tc_row(a, n, r);
    return base + at.t * s[1] + at.h * s[2];
  };
  auto key_at = [&](const T* base, const int64_t (&s)[3], int j) { return key_ok(j) ? base + j * s[1] : nullptr; };
  bool some = false;                         // one of the keys that this thread looked at is there
  auto request = [&](int j, int buf) {
    if (j < j_end) {
      const uint32_t y = ring + buf * kStage, y2 = y + kHalfStage;
      const int e0 = j * kTcOther;
      if constexpr (OWN_ROWS) {
        tc_fetch<T, NP, kTcOther, kTcBwdThreads>(y, a.d, kb, [&](int i) { return key_at(kb, a.ks, e0 + i); });
        tc_fetch<T, NP, kTcOther, kTcBwdThreads>(y2, a.d, vb, [&](int i) { return key_at(vb, a.vs, e0 + i); });
        if (tid < kTcOther) {
          const bool there = key_ok(e0 + tid);
          s_a[buf][tid] = there ? 0.f : -INFINITY;
          some |= there;
        }
      } else {
        tc_fetch<T, NP, kTcOther, kTcBwdThreads>(y, a.d, qb, [&](int i) { return row_at(qb, a.qs, e0 + i); });
        tc_fetch<T, NP, kTcOther, kTcBwdThreads>(y2, a.d, ob, [&](int i) { return row_at(ob, a.os, e0 + i); });
        const int r = e0 + tid % kTcOther;
        if (tid < kTcOther)
          s_a[buf][tid] = r < rows ? -__ldg(a.lse + stat0 + r) : -INFINITY;
        else if (tid < 2 * kTcOther)
          s_b[buf][tid - kTcOther] = r < rows ? -__ldg(a.delta + stat0 + r) : 0.f;
      }
    }
  };
  float own_s;                               // -lse of the thread's query; bias of its key
  const int mine = own0 + lane_id;
  if constexpr (OWN_ROWS) {
    tc_fetch<T, NP, kTcOwn, kTcBwdThreads>(x1, a.d, qb, [&](int i) { return row_at(qb, a.qs, own0 + i); });
    tc_fetch<T, NP, kTcOwn, kTcBwdThreads>(x2, a.d, ob, [&](int i) { return row_at(ob, a.os, own0 + i); });
    request(j_begin, 0);
    own_s = mine < rows ? -__ldg(a.lse + stat0 + mine) : -INFINITY;
    // D: 8 NP threads to a row, 8 channels each, so that a load covers whole lines
    const int c = tid % (8 * NP) * 8;
#pragma unroll
    for (int i = tid / (8 * NP); i < kTcOwn; i += kTcBwdThreads / (8 * NP)) {
      const int r = own0 + i;
      float y = 0.f;
      if (r < rows && c < a.d) {
        const TcRow at = tc_row(a, n, r);
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(ob + at.t * a.os[1] + at.h * a.os[2] + c));
        const float4* o32 = reinterpret_cast<const float4*>(a.out_f32 + ((static_cast<int64_t>(b) * a.Tq + at.t) * a.heads + at.h) * a.d + c);
        const float4 f0 = __ldg(o32), f1 = __ldg(o32 + 1);
        const float2 g0 = tc_unpack<T>(u.x), g1 = tc_unpack<T>(u.y), g2 = tc_unpack<T>(u.z), g3 = tc_unpack<T>(u.w);
        y = fmaf(f0.x, g0.x, fmaf(f0.y, g0.y, fmaf(f0.z, g1.x, f0.w * g1.y)));
        y = fmaf(f1.x, g2.x, fmaf(f1.y, g2.y, fmaf(f1.z, g3.x, fmaf(f1.w, g3.y, y))));
      }
#pragma unroll
      for (int o = 4 * NP; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
      if (c == 0) {
        s_d[i] = y;
        if (r < rows && rank == 0) a.delta[stat0 + r] = y;
      }
    }
  } else {
    tc_fetch<T, NP, kTcOwn, kTcBwdThreads>(x1, a.d, kb, [&](int i) { return key_at(kb, a.ks, own0 + i); });
    tc_fetch<T, NP, kTcOwn, kTcBwdThreads>(x2, a.d, vb, [&](int i) { return key_at(vb, a.vs, own0 + i); });
    request(j_begin, 0);
    own_s = key_ok(mine) ? 0.f : -INFINITY;
  }

  bool ok = tc_landed(true);
  const float own_d = OWN_ROWS ? -s_d[lane_id] : 0.f;
  const float2 c2 = make_float2(a.c, a.c), os2 = make_float2(own_s, own_s), od2 = make_float2(own_d, own_d);
  int it = 0;
  for (int j = j_begin; j < j_end; ++j, ++it) {
    const int buf = it & 1;
    const uint32_t y = ring + buf * kStage, y2 = y + kHalfStage;
    if (it > 0) ok = mbar_wait(&bars[1], (it - 1) & 1);
    if (tid == 0 && ok) {
      tc_fence_after();
      tc_scores<T, NP>(B.tmem + tS, x1, y);
      tc_scores<T, NP>(B.tmem + tD, x2, y2);
      umma_commit(&bars[0]);
    }
    request(j + 1, buf ^ 1);
    ok = __all_sync(0xffffffffu, ok && mbar_wait(&bars[0], it & 1));
    tc_fence_after();
    const uint32_t y_lo = OWN_ROWS ? y2 : ring + 2 * kStage, y2_lo = y_lo + kHalfStage;
    if (ok) {
      if constexpr (kTerms) {
        tc_terms<NP, kTcBwdThreads>(y, y_lo);
        if constexpr (!OWN_ROWS) tc_terms<NP, kTcBwdThreads>(y2, y2_lo);
      }
#pragma unroll
      for (int q = 2 * half; q < 2 * half + 2; ++q) {          // columns 16 q .. 16 q + 15
        uint32_t rs[16], rd[16], ps[16], pd[16];
        tmem_ld_32x32b_x16(B.t_lane + tS + 16 * q, rs);
        tmem_ld_32x32b_x16(B.t_lane + tD + 16 * q, rd);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 sa = *reinterpret_cast<const float2*>(&s_a[buf][16 * q + 2 * i]);
          float2 p = fma2(make_float2(__uint_as_float(rs[2 * i]), __uint_as_float(rs[2 * i + 1])), c2, OWN_ROWS ? sa : os2);
          p = add2(p, OWN_ROWS ? os2 : sa);
          p.x = ex2f(p.x), p.y = ex2f(p.y);
          const float2 dd = OWN_ROWS ? od2 : *reinterpret_cast<const float2*>(&s_b[buf][16 * q + 2 * i]);
          tc_split(mul2(p, add2(make_float2(__uint_as_float(rd[2 * i]), __uint_as_float(rd[2 * i + 1])), dd)), pd, i);
          if constexpr (!OWN_ROWS) tc_split(p, ps, i);
        }
        tmem_st_32x32b_x16(B.t_lane + tD + 16 * q, pd);
        if constexpr (!OWN_ROWS) tmem_st_32x32b_x16(B.t_lane + tS + 16 * q, ps);
      }
      tmem_st_wait();
    }
    ok = tc_landed(ok);
    if (!ok) break;
    if (tid == 0) {
      tc_fence_after();
      tc_sums<NP, kTerms ? 1 : 0>(B.tmem + tA1, B.tmem + tD, y, y_lo, it > 0);
      if constexpr (!OWN_ROWS) tc_sums<NP, kTerms ? 2 : 0>(B.tmem + tA2, B.tmem + tS, y2, y2_lo, it > 0);
      umma_commit(&bars[1]);
    }
  }
  if (ok && it > 0) ok = mbar_wait(&bars[1], (it - 1) & 1);
  tc_fence_after();
  __syncwarp();
  const bool any = it > 0 && (!OWN_ROWS || mask == nullptr || __syncthreads_or(some));   // as in the forward kernel
  const bool gone = !OWN_ROWS && own_s != 0.f;   // a key that is not there: zeros, whatever the queries hold
  const int own_n = OWN_ROWS ? rows : a.Tk;
  auto to_row = [&](void* to, int r) {
    if constexpr (OWN_ROWS) {
      const TcRow at = tc_row(a, n, r);
      return static_cast<T*>(to) + ((static_cast<int64_t>(b) * a.Tq + at.t) * a.heads + at.h) * a.d;
    } else {
      return static_cast<T*>(to) + ((static_cast<int64_t>(b) * a.Tk + r) * a.kv_heads + n) * a.d;
    }
  };
  if (cl > 1) {                              // the operands' memory takes the sums: dq, dk the ring, dv x1 and x2
    cp_async_wait_all();
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < (OWN_ROWS ? 1 : 2); ++k) {
    void* to = OWN_ROWS ? a.dq : k == 0 ? a.dk : a.dv;
    const float f = k == 0 ? a.scale : 1.f;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      float2 v[16];                          // channels 64 p + 32 half ..
      if (any) {
        uint32_t u[32];
        tmem_ld_32x32b_x32(B.t_lane + (k == 0 ? tA1 : tA2) + 64 * p + 32 * half, u);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i)
          v[i] = gone ? make_float2(0.f, 0.f) : make_float2(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1]));
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = make_float2(0.f, 0.f);
      }
      const int c0 = 64 * p + 32 * half;
      if (cl > 1) {
        tc_put<8>((k == 0 ? ring : x1) + p * 2 * kTcTile, lane_id, 8 * half, v, f);
      } else if (mine < own_n && to != nullptr) {
        tc_store_row<T, 4>(to_row(to, mine) + c0, a.d - c0, v, f);
      }
    }
  }
  B.close(kCols);
  if (cl == 1) return;
  cluster_sync_all();
#pragma unroll
  for (int k = 0; k < (OWN_ROWS ? 1 : 2); ++k) {
    void* to = OWN_ROWS ? a.dq : k == 0 ? a.dk : a.dv;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const uint32_t tile = (k == 0 ? ring : x1) + p * 2 * kTcTile;
      for (int i = tid / 16; i * cl + rank < kTcOwn; i += kTcBwdThreads / 16) {
        const int row = i * cl + rank, c = tid % 16, r = own0 + row, at_c = 64 * p + c * 4;
        if (r >= own_n || at_c >= a.d || to == nullptr) continue;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int z = 0; z < cl; ++z) {
          const float4 u = ld_dsmem4(mapa_shared(tc_join_chunk(tile, row, c), z));
          y = make_float4(y.x + u.x, y.y + u.y, y.z + u.z, y.w + u.w);
        }
        *reinterpret_cast<uint2*>(to_row(to, r) + at_c) = make_uint2(tc_pack<T>(y.x, y.y), tc_pack<T>(y.z, y.w));
      }
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
static int xattn_tc_launch(K kernel, PerDeviceOnce& once, const XAttn& a, int own, int other, int threads, int per_sm, int smem,
                           cudaStream_t stream) {
  const int st = allow_smem(once, kernel, smem);
  if (st != SSAM_OK) return st;
  const int tiles = (own + kTcOwn - 1) / kTcOwn;
  const int cl = xattn_tc_cluster(static_cast<int64_t>(a.B) * a.kv_heads * tiles, per_sm, (other + kTcOther - 1) / kTcOther);
  return launch_following(kernel, dim3(tiles * cl, a.kv_heads, a.B), dim3(threads), smem, cl, stream, a);
}

template <class T, int NP>
static int xattn_tc_fwd_t(const XAttn& a, cudaStream_t stream) {
  static PerDeviceOnce once;
  return xattn_tc_launch(xattn_tc_fwd_kernel<T, NP>, once, a, a.group * a.Tq, a.Tk, kTcThreads, 4 / NP,
                         NP * (kTcTile + 4 * kTcHalf) + 1024, stream);
}
template <class T, int NP>
static int xattn_tc_bwd_t(const XAttn& a, cudaStream_t stream) {
  static PerDeviceOnce by_rows, by_keys;
  constexpr int smem = NP * (2 * kTcTile + 4 * kTcHalf) + 1024;
  constexpr int smem_keys = smem + (std::is_same<T, __half>::value ? NP * 2 * kTcHalf : 0);   // the two tiles of remainders
  const int rows = a.group * a.Tq;
  const int st = xattn_tc_launch(xattn_tc_bwd_kernel<T, NP, true>, by_rows, a, rows, a.Tk, kTcBwdThreads, 2 / NP, smem, stream);
  if (st != SSAM_OK || a.dk == nullptr) return st;
  return xattn_tc_launch(xattn_tc_bwd_kernel<T, NP, false>, by_keys, a, a.Tk, rows, kTcBwdThreads, 2 / NP, smem_keys, stream);
}
int xattn_tc(const XAttn& a, int dtype, bool backward, cudaStream_t stream) {
  if (backward) {
    if (a.d <= 64) return dtype == 0 ? xattn_tc_bwd_t<__half, 1>(a, stream) : xattn_tc_bwd_t<__nv_bfloat16, 1>(a, stream);
    return dtype == 0 ? xattn_tc_bwd_t<__half, 2>(a, stream) : xattn_tc_bwd_t<__nv_bfloat16, 2>(a, stream);
  }
  if (a.d <= 64) return dtype == 0 ? xattn_tc_fwd_t<__half, 1>(a, stream) : xattn_tc_fwd_t<__nv_bfloat16, 1>(a, stream);
  return dtype == 0 ? xattn_tc_fwd_t<__half, 2>(a, stream) : xattn_tc_fwd_t<__nv_bfloat16, 2>(a, stream);
}

}  // namespace ssam
