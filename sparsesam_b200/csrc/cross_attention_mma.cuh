// Tensor-core kernels of the cross attention for fp16 / bf16 (formulas and conventions
// in cross_attention.cuh).
//
// Here: one short side (the other case is cross_attention_tc.cu). Everything is built from
// mma.m16n8k16 on registers: the short side is a handful of prompt tokens, so a warp's
// 16-row tile is the whole problem of one head, there is nothing for a 128-row
// tcgen05 tile to share, and DRAM or the exponentials set the pace.
//
// Fragments. With g = lane / 4, t = lane % 4, lane (g, t) of a fragment of 8 token rows
// holds channels t DP/4 .. t DP/4 + DP/4 - 1 of row g: one contiguous load of 8 (DP = 16)
// to 64 bytes. The order in which a product sums over channels is free, so register
// pair s of such a row is used as the k-columns {2t, 2t+1, 2t+8, 2t+9} of 16-channel step
// s for both operands. The second products need the token axis as k: movmatrix turns an
// 8 x 8 block of a fragment, which gives the operand whose column n of block i is channel
// (n / 2) DP/4 + 2 i + n % 2, and a lane's accumulator columns 2t, 2t+1 of block i are
// channels t DP/4 + 2 i, + 1: results leave in the same contiguous DP/4-channel pieces.
//
// Second factors: probabilities and dS are fp32 and enter their product as two half
// terms (value and remainder), so that a result carries one rounding to its type instead
// of two. A single term measured 1.4 times the error of the rounded definition.
//
// fp16 ends at 2^-24, and a key of small weight counts where the larger ones meet zeros.
// So P enters times 2^12 to 2^15, its remainder times another 2^11, in a product of its
// own that joins the first one's sums times 2^-11: 22 bits of every weight down to 2^-26,
// and 2^-48 of the largest at the end. dS has no fixed scale at all (it follows the loss):
// its products run in bf16, which has fp32's range: two bf16 terms of dS, the fp16 factor
// as two bf16 terms (exact, 11 bits = 8 + 3), without the product of the two remainders.
#pragma once

#include "cross_attention.cuh"

namespace ssam {

template <class T>
struct Mma;
template <>
struct Mma<__half> {
  static __device__ __forceinline__ void run(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ void run8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(b0));
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }
};
template <>
struct Mma<__nv_bfloat16> {
  static __device__ __forceinline__ void run(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ void run8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(b0));
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) { return pack_bf16x2(x, y); }
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
};

__device__ __forceinline__ void store1(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store1(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ uint32_t movm(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// x, y -> packed value and packed remainder
template <class T>
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = Mma<T>::pack(x, y);
  const float2 h = Mma<T>::unpack(hi), r = add2(make_float2(x, y), make_float2(-h.x, -h.y));
  lo = Mma<T>::pack(r.x, r.y);
}

template <class T>
constexpr bool kIsHalf = false;
template <>
constexpr bool kIsHalf<__half> = true;

// P, scaled, as two terms of T: the remainder of fp16 in units of 2^-11
template <class T>
__device__ __forceinline__ void p_terms(float x, float y, uint32_t& hi, uint32_t& lo) {
  if constexpr (kIsHalf<T>) {
    hi = Mma<T>::pack(x, y);
    const float2 h = Mma<T>::unpack(hi), r = mul2(add2(make_float2(x, y), make_float2(-h.x, -h.y)), make_float2(2048.f, 2048.f));
    lo = Mma<T>::pack(r.x, r.y);
  } else {
    split2<T>(x, y, hi, lo);
  }
}
// acc (the remainders' product so far) in units of the values
template <class T>
__device__ __forceinline__ void lo_to_hi(float (&acc)[4]) {
  if constexpr (kIsHalf<T>) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] *= 1.f / 2048.f;
  }
}

// This lane's DP / 4 channels of a token row (DP / 8 registers); zeros past channel d and when !ok.
template <class T, int DP>
__device__ __forceinline__ void load_frag(const T* row, int t, int d, bool ok, uint32_t (&r)[DP / 8]) {
  const T* p = row + t * (DP / 4);
  if constexpr (DP == 16) {
    uint2 u = make_uint2(0u, 0u);
    if (ok && t * 4 < d) u = __ldg(reinterpret_cast<const uint2*>(p));
    r[0] = u.x, r[1] = u.y;
  } else {
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) {
      uint4 u = make_uint4(0u, 0u, 0u, 0u);
      if (ok && t * (DP / 4) + i * 8 < d) u = __ldg(reinterpret_cast<const uint4*>(p + i * 8));
      r[4 * i] = u.x, r[4 * i + 1] = u.y, r[4 * i + 2] = u.z, r[4 * i + 3] = u.w;
    }
  }
}
// Stores a lane's DP / 4 channels (packed pairs) of a row.
template <class T, int DP>
__device__ __forceinline__ void store_frag(T* row, int t, int d, const uint32_t (&r)[DP / 8]) {
  T* p = row + t * (DP / 4);
  if constexpr (DP == 16) {
    if (t * 4 < d) *reinterpret_cast<uint2*>(p) = make_uint2(r[0], r[1]);
  } else {
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
      if (t * (DP / 4) + i * 8 < d)
        *reinterpret_cast<uint4*>(p + i * 8) = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
  }
}

constexpr int kXmWarps = 8;
constexpr int kXmThreads = 32 * kXmWarps;
// Blocks per SM that the forward kernels' registers are held to, and may use up to: N tiles of 8 entries of the short side
// in registers (S = 2: keys, half the accumulators of rows), DP channels. These are the blocks that fit without a word
// to the compiler, which then leaves registers unused (24 x 4096 of 64 channels, 64 images: 74 us, 70 so; 4096 x 13 of 16
// 39.4 and 37.9) or, a few past the border, a block (64 x 4096 of 16, fp16).
template <int DP, int N, int S>
constexpr int kXmBlocks = DP * N <= 16 * S ? 2 + S : DP * N <= 32 * S && S == 2 && DP <= 32 ? 3 : DP * N <= 64 * S && DP <= 64 ? 2 : 1;

// Query row r of key head n -> element offset
__device__ __forceinline__ int64_t row_offset(const XAttn& a, const int64_t (&st)[3], int b, int n, int r) {
  if (a.group == 1) return b * st[0] + r * st[1] + n * st[2];
  const int g = r / a.Tq, t = r - g * a.Tq;
  return b * st[0] + t * st[1] + (n * a.group + g) * st[2];
}
// the same into contiguous [B, Tq, heads, d]
__device__ __forceinline__ int64_t row_dense(const XAttn& a, int b, int n, int r) {
  const int g = a.group == 1 ? 0 : r / a.Tq, t = r - g * a.Tq;
  return ((static_cast<int64_t>(b) * a.Tq + t) * a.heads + n * a.group + g) * a.d;
}

constexpr float kXmNone = -3.402823466e38f;  // reference before the first key: no finite logit is below it
// The reference is kXmBelow<T> below the maximum that it was taken at, and renewed when a logit is kXmSlack<T> above it:
// exponentials end at 2^8, for fp16 at 2^15, of which 2^12 is the scale of its terms.
template <class T>
constexpr float kXmBelow = kIsHalf<T> ? 12.f : 0.f;
template <class T>
constexpr float kXmSlack = kIsHalf<T> ? 15.f : 8.f;

// ---------------------------------------------------------------------------
// Forward, few query rows (8 NQ per block) on many keys. The short side is the column
// side, S^T = K Q^T (16 keys x 8 queries per instruction: no padding rows for the
// decoder's 8 tokens), and O^T = V^T P^T. The keys are split over the block's warps and
// the cluster; nothing passes between warps until the end.
//
// The reference point of the exponentials is renewed only when a logit exceeds it by
// 2^8 (as in attention.cu), so the cross-lane maximum is not taken every step.
//
// HP = 2 (heads of 16 next to one another): a fragment is two heads of a token, 64 contiguous
// bytes, because 32-byte pieces keep the L1 tags, not the DRAM, busy (tokens -> image, 64 images:
// 35 us with HP = 1 at 72 % of L1, 26.4 with HP = 2 at 5.1 TB/s; one image 4.5 us, a launch and a join). Lanes t < 2 hold the first head's channels, so key
// and query fragments with the other half zeroed (both: 0 times a NaN of the other head is one) give one head's
// logits. V^T rows g < 4 are the first head's; each head has accumulators of its own, and half of their rows count.
// Twice the tensor instructions, of which there are plenty.
// ---------------------------------------------------------------------------
template <class T, int DP, int NQ, int HP>
__global__ void __launch_bounds__(kXmThreads, kXmBlocks<DP, HP * NQ, 1>) xattn_fwd_few_rows(const XAttn args, int) {
  const XAttn a = follow(args, args.lse == nullptr);
  constexpr int NR = DP / 8, NU = NR / 2;    // 8- and 16-channel blocks
  constexpr int KM = DP <= 32 && HP * NQ <= 4 ? 2 : 1;   // 16-key tiles per step
  extern __shared__ __align__(16) float xsm[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int b = blockIdx.z, n = blockIdx.y * HP;
  const int cl = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
  const int rows = a.group * a.Tq;
  const int r0 = static_cast<int>(blockIdx.x) / cl * 8 * NQ;
  const int keys = xattn_keys(a, b);
  const int steps = (keys + 16 * KM - 1) / (16 * KM), ns = kXmWarps * cl;
  const int per = (steps + ns - 1) / ns * (16 * KM);
  const int j_begin = min(keys, (rank * kXmWarps + warp) * per), j_end = min(keys, j_begin + per);
  const uint8_t* mask = a.key_mask == nullptr ? nullptr : a.key_mask + static_cast<int64_t>(b) * a.Tk;
  const int d = HP * a.d;                    // channels of a fragment
  const T* kp = static_cast<const T*>(a.k) + b * a.ks[0] + n * a.ks[2] + (j_begin + g) * a.ks[1];
  const T* vp = static_cast<const T*>(a.v) + b * a.vs[0] + n * a.vs[2] + (j_begin + g) * a.vs[1];

  uint32_t k[KM][2][NR], v[KM][2][NR];
  float bias[KM][2];                         // 0, or -infinity for a key that is not there
  bool some = false;                         // of this lane's keys one is there
  auto load = [&](int j0) {                  // loads keys j0 + .. and moves on
    if (mask == nullptr && j0 + 16 * KM <= j_end) {
      some = true;
#pragma unroll
      for (int i = 0; i < 2 * KM; ++i) {
        bias[i / 2][i % 2] = 0.f;
        load_frag<T, DP>(kp + i * 8 * a.ks[1], t, d, true, k[i / 2][i % 2]);
        load_frag<T, DP>(vp + i * 8 * a.vs[1], t, d, true, v[i / 2][i % 2]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2 * KM; ++i) {
        const int j = j0 + i * 8 + g;
        const bool ok = j < j_end && (mask == nullptr || __ldg(mask + j) != 0);
        some |= ok;
        bias[i / 2][i % 2] = ok ? 0.f : -INFINITY;
        load_frag<T, DP>(kp + i * 8 * a.ks[1], t, d, ok, k[i / 2][i % 2]);
        load_frag<T, DP>(vp + i * 8 * a.vs[1], t, d, ok, v[i / 2][i % 2]);
      }
    }
    kp += 16 * KM * a.ks[1];
    vp += 16 * KM * a.vs[1];
  };
  load(j_begin);
  uint32_t q[HP][NQ][NR];
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    const int r = r0 + i * 8 + g;
    uint32_t x[NR];
    load_frag<T, DP>(static_cast<const T*>(a.q) + row_offset(a, a.qs, b, n, min(r, rows - 1)), t, d, r < rows, x);
#pragma unroll
    for (int z = 0; z < HP; ++z)
#pragma unroll
      for (int c = 0; c < NR; ++c) q[z][i][c] = HP == 1 || t / 2 == z ? x[c] : 0u;
  }
  float o[HP][NQ][NU][4];
  float2 ref[HP][NQ], l[HP][NQ];             // of queries 2t, 2t + 1
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
#pragma unroll
    for (int z = 0; z < HP; ++z) {
      ref[z][i] = make_float2(kXmNone, kXmNone), l[z][i] = make_float2(0.f, 0.f);
#pragma unroll
      for (int u = 0; u < NU; ++u) o[z][i][u][0] = o[z][i][u][1] = o[z][i][u][2] = o[z][i][u][3] = 0.f;
    }
  }
  const float2 c2 = make_float2(a.c, a.c);

  for (int j0 = j_begin; j0 < j_end; j0 += 16 * KM) {
    float2 s[HP][NQ][KM][2];                 // [key g | g + 8] x queries 2t, 2t + 1
    uint32_t vt[KM][2][NR];
    bool renew = false;
#pragma unroll
    for (int x = 0; x < KM; ++x) {
#pragma unroll
      for (int z = 0; z < HP; ++z) {
        uint32_t kz[2][NR];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int c = 0; c < NR; ++c) kz[h][c] = HP == 1 || t / 2 == z ? k[x][h][c] : 0u;
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
          float f[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < NR; c += 2)
            Mma<T>::run(f, kz[0][c], kz[1][c], kz[0][c + 1], kz[1][c + 1], q[z][i][c], q[z][i][c + 1]);
#pragma unroll
          for (int h = 0; h < 2; ++h)
            s[z][i][x][h] = fma2(make_float2(f[2 * h], f[2 * h + 1]), c2, make_float2(bias[x][h], bias[x][h]));
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < NR; ++c) vt[x][h][c] = movm(v[x][h][c]);
    }
    if (j0 + 16 * KM < j_end) load(j0 + 16 * KM);     // the next step's, under this one's arithmetic
#pragma unroll
    for (int z = 0; z < HP; ++z)
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        float2 m = ref[z][i];
#pragma unroll
        for (int x = 0; x < KM; ++x)
#pragma unroll
          for (int h = 0; h < 2; ++h) m.x = fmaxf(m.x, s[z][i][x][h].x), m.y = fmaxf(m.y, s[z][i][x][h].y);
        renew |= m.x > ref[z][i].x + kXmSlack<T> || m.y > ref[z][i].y + kXmSlack<T>;
      }
    if (__any_sync(0xffffffffu, renew)) {
#pragma unroll
      for (int i = 0; i < NQ; ++i)
#pragma unroll
        for (int z = 0; z < HP; ++z) {
          float2 m = ref[z][i];
#pragma unroll
          for (int x = 0; x < KM; ++x)
#pragma unroll
            for (int h = 0; h < 2; ++h) m.x = fmaxf(m.x, s[z][i][x][h].x), m.y = fmaxf(m.y, s[z][i][x][h].y);
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) {
            m.x = fmaxf(m.x, __shfl_xor_sync(0xffffffffu, m.x, w));
            m.y = fmaxf(m.y, __shfl_xor_sync(0xffffffffu, m.y, w));
          }
          // not below the old one: the other queries' renewals must not lower it
          m.x = fmaxf(m.x - kXmBelow<T>, ref[z][i].x), m.y = fmaxf(m.y - kXmBelow<T>, ref[z][i].y);
          const float2 f = make_float2(ex2f(ref[z][i].x - m.x), ex2f(ref[z][i].y - m.y));
          ref[z][i] = m;
          l[z][i] = mul2(l[z][i], f);
#pragma unroll
          for (int u = 0; u < NU; ++u) o[z][i][u][0] *= f.x, o[z][i][u][1] *= f.y, o[z][i][u][2] *= f.x, o[z][i][u][3] *= f.y;
        }
    }
#pragma unroll
    for (int x = 0; x < KM; ++x) {
      uint32_t hi[HP][NQ][2], lo[HP][NQ][2];
#pragma unroll
      for (int z = 0; z < HP; ++z)
#pragma unroll
        for (int i = 0; i < NQ; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float2 p = add2(s[z][i][x][h], make_float2(-ref[z][i].x, -ref[z][i].y));
            p.x = ex2f(p.x), p.y = ex2f(p.y);
            l[z][i] = add2(l[z][i], p);
            p_terms<T>(p.x, p.y, hi[z][i][h], lo[z][i][h]);
            hi[z][i][h] = movm(hi[z][i][h]), lo[z][i][h] = movm(lo[z][i][h]);
          }
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int z = 0; z < HP; ++z)
#pragma unroll
          for (int i = 0; i < NQ; ++i) {
            float(&acc)[4] = o[z][i][u];
            const uint32_t(&va)[2][NR] = vt[x];
            if constexpr (kIsHalf<T>) {
              float rest[4] = {0.f, 0.f, 0.f, 0.f};
              Mma<T>::run(rest, va[0][2 * u], va[0][2 * u + 1], va[1][2 * u], va[1][2 * u + 1], lo[z][i][0], lo[z][i][1]);
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[e] = fmaf(rest[e], 1.f / 2048.f, acc[e]);
            } else {
              Mma<T>::run(acc, va[0][2 * u], va[0][2 * u + 1], va[1][2 * u], va[1][2 * u + 1], lo[z][i][0], lo[z][i][1]);
            }
            Mma<T>::run(acc, va[0][2 * u], va[0][2 * u + 1], va[1][2 * u], va[1][2 * u + 1], hi[z][i][0], hi[z][i][1]);
          }
    }
  }

  if (!__any_sync(0xffffffffu, some)) {      // a query that is not finite leaves NaN here, which is nothing's
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
#pragma unroll
      for (int z = 0; z < HP; ++z) {
        ref[z][i] = make_float2(kXmNone, kXmNone), l[z][i] = make_float2(0.f, 0.f);
#pragma unroll
        for (int u = 0; u < NU; ++u) o[z][i][u][0] = o[z][i][u][1] = o[z][i][u][2] = o[z][i][u][3] = 0.f;
      }
    }
  }

  // Join. Every warp leaves its references and sums; the block joins them at their highest reference, and
  // the cluster's blocks theirs on the way out, in a fixed order.
  constexpr int PER = NU * 4 + 2, NREG = NQ * PER, ROWS = HP * 8 * NQ;
  float* s_ref = xsm;                        // [8][ROWS]: head z, query 8 i + x at z 8 NQ + 8 i + x
  float* s_top = s_ref + kXmWarps * ROWS;    // [ROWS]
  float* s_acc = s_top + ROWS;               // [8][NREG][32]; the block's sums end up in [0]
  const int hz = HP == 1 ? 0 : g / 4;        // the head of this lane's sums
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    float* to = s_acc + (warp * NREG + i * PER) * 32 + lane;
#pragma unroll
    for (int z = 0; z < HP; ++z) {
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) {
        l[z][i].x += __shfl_xor_sync(0xffffffffu, l[z][i].x, w);
        l[z][i].y += __shfl_xor_sync(0xffffffffu, l[z][i].y, w);
      }
      if (g == 0) *reinterpret_cast<float2*>(s_ref + warp * ROWS + (z * NQ + i) * 8 + 2 * t) = ref[z][i];
      if (HP == 1 || hz == z) to[NU * 4 * 32] = l[z][i].x, to[(NU * 4 + 1) * 32] = l[z][i].y;
    }
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) to[(u * 4 + e) * 32] = hz == 0 ? o[0][i][u][e] : o[HP - 1][i][u][e];
  }
  __syncthreads();
  for (int w = warp; w < NREG; w += kXmWarps) {          // register w of every lane; its query is 8 i + 2t + (w & 1)
    const int ro = (hz * NQ + w / PER) * 8 + 2 * t + (w % PER & 1);
    float top = kXmNone, x = 0.f;
#pragma unroll
    for (int z = 0; z < kXmWarps; ++z) top = fmaxf(top, s_ref[z * ROWS + ro]);
#pragma unroll
    for (int z = 0; z < kXmWarps; ++z) x = fmaf(s_acc[(z * NREG + w) * 32 + lane], ex2f(s_ref[z * ROWS + ro] - top), x);
    s_acc[w * 32 + lane] = x;                            // read by this lane only so far
    if (w % PER < 2 && g % (8 / HP) == 0) s_top[ro] = top;
  }
  if (cl > 1) cluster_sync_all(); else __syncthreads();
  const uint32_t base = smem_u32(s_acc) + lane * 4;
  const int64_t stat0 = (static_cast<int64_t>(b) * a.heads + (n + hz) * a.group) * a.Tq;
  for (int w = rank * kXmWarps + warp; w < 2 * NQ * NU; w += cl * kXmWarps) {
    const int e = w % 2, u = w / 2 % NU, i = w / 2 / NU, ro = (hz * NQ + i) * 8 + 2 * t + e, r = r0 + i * 8 + 2 * t + e;
    float x = 0.f, y = 0.f, den = 0.f, m = kXmNone;
    for (int z = 0; z < cl; ++z) m = fmaxf(m, ld_dsmem(mapa_shared(smem_u32(s_top + ro), z)));
    for (int z = 0; z < cl; ++z) {
      const uint32_t from = mapa_shared(base, z);
      const float f = ex2f(ld_dsmem(mapa_shared(smem_u32(s_top + ro), z)) - m);
      x = fmaf(ld_dsmem(from + (i * PER + u * 4 + e) * 128), f, x);
      y = fmaf(ld_dsmem(from + (i * PER + u * 4 + e + 2) * 128), f, y);
      den = fmaf(ld_dsmem(from + (i * PER + NU * 4 + e) * 128), f, den);
    }
    if (r >= rows) continue;
    const float inv = den == 0.f ? 0.f : 1.f / den;
    const int ch = g / 2 % (4 / HP) * (DP / 4) + 4 * u + g % 2;   // and ch + 2, of head n + hz
    T* to = static_cast<T*>(a.out) + row_offset(a, a.os, b, n + hz, r);
    float* to32 = a.out_f32 == nullptr ? nullptr : a.out_f32 + row_dense(a, b, n + hz, r);
    if (ch < a.d) {
      store1(to + ch, x * inv);
      if (to32 != nullptr) to32[ch] = x * inv;
    }
    if (ch + 2 < a.d) {
      store1(to + ch + 2, y * inv);
      if (to32 != nullptr) to32[ch + 2] = y * inv;
    }
    if (a.lse != nullptr && u == 0 && g % (8 / HP) == 0) a.lse[stat0 + r] = den == 0.f ? INFINITY : m + log2f(den);
  }
  if (cl > 1) cluster_sync_all();
}

// ---------------------------------------------------------------------------
// Forward, many queries on few keys (at most 8 NK): a warp keeps the K and turned V
// fragments of one (image, query head) and walks its share of the queries 16 at a time, the
// next rows in flight. 64 images, 4096 queries on 8 keys: 32 us, 4.2 TB/s, issuing in 69 % of the cycles; neighbouring warps hold neighbouring heads, so a block touches whole rows. HP = 2 as above.
// ---------------------------------------------------------------------------
template <class T, int DP, int NK, int HP>
__global__ void __launch_bounds__(kXmThreads, kXmBlocks<DP, HP * NK, 2>) xattn_fwd_few_keys(const XAttn args, int chunks) {
  const XAttn a = follow(args, false);
  constexpr int NR = DP / 8;
  constexpr float kP = kIsHalf<T> ? 16384.f : 1.f;       // P is at most 1
  const int lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int units = a.heads / HP;
  const int64_t w = static_cast<int64_t>(blockIdx.x) * kXmWarps + threadIdx.x / 32;
  const int h = static_cast<int>(w % units) * HP, chunk = static_cast<int>(w / units % chunks);
  const int64_t bb = w / units / chunks;
  if (bb >= a.B) return;
  const int b = static_cast<int>(bb), n = h / a.group;
  const int tiles = (a.Tq + 15) / 16, per = (tiles + chunks - 1) / chunks;
  const int r_begin = min(a.Tq, chunk * per * 16), r_end = min(a.Tq, r_begin + per * 16);
  if (r_begin >= r_end) return;
  const int keys = xattn_keys(a, b), d = HP * a.d;
  const T* kb = static_cast<const T*>(a.k) + b * a.ks[0] + n * a.ks[2];
  const T* vb = static_cast<const T*>(a.v) + b * a.vs[0] + n * a.vs[2];
  const uint8_t* mask = a.key_mask == nullptr ? nullptr : a.key_mask + static_cast<int64_t>(b) * a.Tk;
  // rows r0 + g and r0 + g + 8
  const T* qp = static_cast<const T*>(a.q) + b * a.qs[0] + h * a.qs[2] + static_cast<int64_t>(r_begin + g) * a.qs[1];
  T* op = static_cast<T*>(a.out) + b * a.os[0] + h * a.os[2] + static_cast<int64_t>(r_begin + g) * a.os[1];
  const int64_t q8 = 8 * a.qs[1], o8 = 8 * a.os[1];
  float* lse = a.lse == nullptr ? nullptr : a.lse + (static_cast<int64_t>(b) * a.heads + h) * a.Tq;
  float* o32 = a.out_f32 == nullptr ? nullptr : a.out_f32 + (static_cast<int64_t>(b) * a.Tq * a.heads + h) * a.d + t * (DP / 4);

  uint32_t k[HP][NK][NR], v[NK][NR], q[2][NR];
  float2 bias[NK];                           // of keys 8 i + 2t, + 1
  int q_end = r_end;                         // rows past it are zeros
  auto load_q = [&](int r) {
    load_frag<T, DP>(qp, t, d, r + g < q_end, q[0]);
    load_frag<T, DP>(qp + q8, t, d, r + g + 8 < q_end, q[1]);
    qp += 2 * q8;
  };
  load_q(r_begin);
  bool some = false;
#pragma unroll
  for (int i = 0; i < NK; ++i) {
    const int j = i * 8 + g;
    const bool ok = j < keys && (mask == nullptr || __ldg(mask + j) != 0);
    some |= ok;
    uint32_t x[NR], y[NR];
    load_frag<T, DP>(kb + j * a.ks[1], t, d, ok, x);
    load_frag<T, DP>(vb + j * a.vs[1], t, d, ok, y);
    const float mine = ok ? 0.f : -INFINITY;
    bias[i].x = __shfl_sync(0xffffffffu, mine, 8 * t);
    bias[i].y = __shfl_sync(0xffffffffu, mine, 8 * t + 4);
#pragma unroll
    for (int c = 0; c < NR; ++c) {
      v[i][c] = movm(y[c]);
#pragma unroll
      for (int z = 0; z < HP; ++z) k[z][i][c] = HP == 1 || t / 2 == z ? x[c] : 0u;
    }
  }

  if (!__any_sync(0xffffffffu, some)) {      // no keys: whatever the queries hold, their rows are zeros
    q_end = r_begin;
#pragma unroll
    for (int c = 0; c < NR; ++c) q[0][c] = q[1][c] = 0u;
  }

  const float2 c2 = make_float2(a.c, a.c);
  for (int r0 = r_begin; r0 < r_end; r0 += 16) {
    float2 s[HP][NK][2];
#pragma unroll
    for (int z = 0; z < HP; ++z) {
      uint32_t qz[2][NR];
#pragma unroll
      for (int c = 0; c < NR; ++c) {
        qz[0][c] = HP == 1 || t / 2 == z ? q[0][c] : 0u;
        qz[1][c] = HP == 1 || t / 2 == z ? q[1][c] : 0u;
      }
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        float f[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NR; c += 2) Mma<T>::run(f, qz[0][c], qz[1][c], qz[0][c + 1], qz[1][c + 1], k[z][i][c], k[z][i][c + 1]);
        s[z][i][0] = fma2(make_float2(f[0], f[1]), c2, bias[i]);
        s[z][i][1] = fma2(make_float2(f[2], f[3]), c2, bias[i]);
      }
    }
    if (r0 + 16 < r_end) load_q(r0 + 16);
    float m[HP][2], l[HP][2];
    float o[HP][NR][4];
#pragma unroll
    for (int z = 0; z < HP; ++z) {
#pragma unroll
      for (int c = 0; c < NR; ++c) o[z][c][0] = o[z][c][1] = o[z][c][2] = o[z][c][3] = 0.f;
      float inv[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = kXmNone;                   // a row without keys: 2^(-inf + 3.4e38) = 0
#pragma unroll
        for (int i = 0; i < NK; ++i) x = fmaxf(x, fmaxf(s[z][i][e].x, s[z][i][e].y));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
        m[z][e] = x;
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < NK; ++i) {
          float2 p = add2(s[z][i][e], make_float2(-x, -x));
          p.x = ex2f(p.x), p.y = ex2f(p.y);
          s[z][i][e] = p;
          sum = add2(sum, p);
        }
        float y = sum.x + sum.y;
        y += __shfl_xor_sync(0xffffffffu, y, 1);
        y += __shfl_xor_sync(0xffffffffu, y, 2);
        l[z][e] = y;
        inv[e] = y == 0.f ? 0.f : kP * rcp_fast(y);
      }
      constexpr int PAIR = NK > 1 ? 2 : 1;
      uint32_t hi[NK / PAIR][4], lo[NK / PAIR][4];
#pragma unroll
      for (int i = 0; i < NK; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 p = mul2(s[z][i][e], make_float2(inv[e], inv[e]));
          p_terms<T>(p.x, p.y, hi[i / PAIR][2 * (i % PAIR) + e], lo[i / PAIR][2 * (i % PAIR) + e]);
        }
#pragma unroll
      for (int c = 0; c < NR; ++c) {
        float(&acc)[4] = o[z][c];
        if constexpr (NK == 1) {
          Mma<T>::run8(acc, lo[0][0], lo[0][1], v[0][c]);
          lo_to_hi<T>(acc);
          Mma<T>::run8(acc, hi[0][0], hi[0][1], v[0][c]);
        } else {
#pragma unroll
          for (int i = 0; i < NK / 2; ++i) Mma<T>::run(acc, lo[i][0], lo[i][1], lo[i][2], lo[i][3], v[2 * i][c], v[2 * i + 1][c]);
          lo_to_hi<T>(acc);
#pragma unroll
          for (int i = 0; i < NK / 2; ++i) Mma<T>::run(acc, hi[i][0], hi[i][1], hi[i][2], hi[i][3], v[2 * i][c], v[2 * i + 1][c]);
        }
      }
    }
    // lane t's columns are channels of head t / 2 of a pair
    if constexpr (HP == 2) {
#pragma unroll
      for (int c = 0; c < NR; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[0][c][e] = t / 2 == 0 ? o[0][c][e] : o[1][c][e];
    }
    if constexpr (kIsHalf<T>) {
#pragma unroll
      for (int c = 0; c < NR; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[0][c][e] *= 1.f / kP;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = r0 + e * 8 + g;
      if (r >= r_end) continue;
      uint32_t y[NR];
#pragma unroll
      for (int c = 0; c < NR; ++c) y[c] = Mma<T>::pack(o[0][c][2 * e], o[0][c][2 * e + 1]);
      store_frag<T, DP>(op + e * o8, t, d, y);
      if (lse != nullptr && t < HP) {
        const float ml = HP == 2 && t == 1 ? m[HP - 1][e] : m[0][e], ll = HP == 2 && t == 1 ? l[HP - 1][e] : l[0][e];
        lse[static_cast<int64_t>(t) * a.Tq + r] = ll == 0.f ? INFINITY : ml + log2f(ll);
      }
      if (o32 != nullptr) {
        float* f = o32 + static_cast<int64_t>(r) * a.heads * a.d;
#pragma unroll
        for (int c = 0; c < NR; ++c)
          if (t * (DP / 4) + 2 * c < d) *reinterpret_cast<float2*>(f + 2 * c) = make_float2(o[0][c][2 * e], o[0][c][2 * e + 1]);
      }
    }
    op += 2 * o8;
  }
}

// ---------------------------------------------------------------------------
// Backward, with p = 2^(c s - lse) and ds = p (dp - D). P is at most 1.
// ---------------------------------------------------------------------------
template <class T>
constexpr float kPScale = kIsHalf<T> ? 16384.f : 1.f;

// Turned blocks of N fragments of 8 tokens (tokens become the k axis), as bf16 for the dS products
template <class T, int N, int NR>
struct Turned {
  uint32_t hi[N][NR], lo[kIsHalf<T> ? N : 1][kIsHalf<T> ? NR : 1];
  __device__ __forceinline__ void make(const uint32_t (&x)[N][NR]) {
#pragma unroll
    for (int h = 0; h < N; ++h)
#pragma unroll
      for (int c = 0; c < NR; ++c) {
        if constexpr (kIsHalf<T>) {
          const float2 f = Mma<__half>::unpack(x[h][c]);
          uint32_t vh, vl;
          split2<__nv_bfloat16>(f.x, f.y, vh, vl);
          hi[h][c] = movm(vh), lo[h][c] = movm(vl);
        } else {
          hi[h][c] = movm(x[h][c]);
        }
      }
  }
};
// acc[c] += (hi + lo)[16 x 16] y[16 x 8 NR], y = tiles y0, y0 + 1
template <class T, int N, int NR>
__device__ __forceinline__ void ds_product(float (&acc)[NR][4], const uint32_t (&hi)[4], const uint32_t (&lo)[4],
                                           const Turned<T, N, NR>& y, int y0) {
  using B = Mma<__nv_bfloat16>;
#pragma unroll
  for (int c = 0; c < NR; ++c) {
    B::run(acc[c], hi[0], hi[1], hi[2], hi[3], y.hi[y0][c], y.hi[y0 + 1][c]);
    B::run(acc[c], lo[0], lo[1], lo[2], lo[3], y.hi[y0][c], y.hi[y0 + 1][c]);
    if constexpr (kIsHalf<T>) B::run(acc[c], hi[0], hi[1], hi[2], hi[3], y.lo[y0][c], y.lo[y0 + 1][c]);
  }
}

// Sum over a row's channels of dout * out (fp32), for the row of this lane's fragment; all t lanes get it.
template <class T, int DP>
__device__ __forceinline__ float row_delta(const float* o32, const uint32_t (&x)[DP / 8], int t, int d, bool ok) {
  float f = 0.f;
  if (ok) {
#pragma unroll
    for (int c = 0; c < DP / 8; ++c) {
      if (t * (DP / 4) + 2 * c >= d) break;
      const float2 o = __ldg(reinterpret_cast<const float2*>(o32 + t * (DP / 4) + 2 * c)), y = Mma<T>::unpack(x[c]);
      f = fmaf(o.x, y.x, f);
      f = fmaf(o.y, y.y, f);
    }
  }
  f += __shfl_xor_sync(0xffffffffu, f, 1);
  return f + __shfl_xor_sync(0xffffffffu, f, 2);
}

// One short side: its 8 NF entries ("few") are all of it, the columns of every tile, and stay in
// registers with their gradient sums; warps and cluster share the long side, 16 entries at a time,
// whose gradients are complete at once and leave at once. One pass over all inputs: 64 images, 8 queries on
// 4096 keys, with the forward pass 108 us; 2.5 TB/s.
//   few = query rows (FEW_ROWS): x = k, v;  y = q, dout.  dk = ds y1, dv = p y2 leave;  dq^T += k^T ds stays
//   few = keys:                  x = q, dout;  y = k, v.  dq = ds y1 leaves;  dk^T += q^T ds, dv^T += dout^T p stay
template <class T, int DP, int NF, bool FEW_ROWS>
__global__ void __launch_bounds__(kXmThreads) xattn_bwd_few(const XAttn args, int) {
  const XAttn a = follow(args, false);
  constexpr int NR = DP / 8, NU = NR / 2;
  constexpr float kP = kPScale<T>;
  using B16 = Mma<__nv_bfloat16>;
  extern __shared__ __align__(16) float xsm[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int b = blockIdx.z, n = blockIdx.y;
  const int cl = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
  const int rows = a.group * a.Tq, keys = xattn_keys(a, b);
  const T* qb = static_cast<const T*>(a.q);
  const T* ob = static_cast<const T*>(a.dout);
  const T* kb = static_cast<const T*>(a.k) + b * a.ks[0] + n * a.ks[2];
  const T* vb = static_cast<const T*>(a.v) + b * a.vs[0] + n * a.vs[2];
  const uint8_t* mask = a.key_mask == nullptr ? nullptr : a.key_mask + static_cast<int64_t>(b) * a.Tk;
  const int64_t stat0 = (static_cast<int64_t>(b) * a.heads + n * a.group) * a.Tq;
  auto key_ok = [&](int j) { return j < keys && (mask == nullptr || __ldg(mask + j) != 0); };
  auto load_row = [&](int r, int end, uint32_t(&x1)[NR], uint32_t(&x2)[NR]) {
    const int rr = min(r, rows - 1);
    load_frag<T, DP>(qb + row_offset(a, a.qs, b, n, rr), t, a.d, r < end, x1);
    load_frag<T, DP>(ob + row_offset(a, a.os, b, n, rr), t, a.d, r < end, x2);
  };
  auto load_key = [&](int j, bool ok, uint32_t(&x1)[NR], uint32_t(&x2)[NR]) {
    load_frag<T, DP>(kb + j * a.ks[1], t, a.d, ok, x1);
    load_frag<T, DP>(vb + j * a.vs[1], t, a.d, ok, x2);
  };

  // few = rows: every key's gradient is written, the zeros of those that are not there too
  const int total = FEW_ROWS ? a.Tk : rows;
  const int steps = (total + 15) / 16, ns = kXmWarps * cl, per = (steps + ns - 1) / ns * 16;
  const int begin = min(total, (rank * kXmWarps + warp) * per), end = min(total, begin + per);
  uint32_t x1[2][NR], x2[2][NR];
  float xs[2], xd[2];                        // long keys: bias of the key; long rows: maximum and D, found below
  bool some = false;                         // of this lane's keys one is there
  int row_end = end;                         // long rows past it are zeros
  auto load_long = [&](int i0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = i0 + h * 8 + g;
      if constexpr (FEW_ROWS) {
        const bool ok = i < end && key_ok(i);
        load_key(i, ok, x1[h], x2[h]);
        xs[h] = ok ? 0.f : -INFINITY;
        some |= ok;
      } else {
        load_row(i, row_end, x1[h], x2[h]);
      }
    }
  };
  load_long(begin);

  uint32_t y1[NF][NR], y2[NF][NR];
  float fs[NF][2], fd[NF][2];                // of few entries 8 i + 2t + e: lse and D of rows; bias of keys
#pragma unroll
  for (int i = 0; i < NF; ++i) {
    const int f = i * 8 + g;
    float mine, del = 0.f;
    if constexpr (FEW_ROWS) {
      load_row(f, rows, y1[i], y2[i]);
      mine = f < rows ? __ldg(a.lse + stat0 + f) : INFINITY;
      del = row_delta<T, DP>(a.out_f32 + row_dense(a, b, n, min(f, rows - 1)), y2[i], t, a.d, f < rows);
    } else {
      const bool ok = key_ok(f);
      load_key(f, ok, y1[i], y2[i]);
      mine = ok ? 0.f : -INFINITY;
      some |= ok;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      fs[i][e] = __shfl_sync(0xffffffffu, mine, 8 * t + 4 * e);
      fd[i][e] = __shfl_sync(0xffffffffu, del, 8 * t + 4 * e);
    }
  }
  if constexpr (!FEW_ROWS) {
    if (!__any_sync(0xffffffffu, some)) {    // no keys: whatever the rows hold, their gradients are zeros
      row_end = begin;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < NR; ++c) x1[h][c] = x2[h][c] = 0u;
    }
  }
  Turned<T, NF, NR> y1t;
  y1t.make(y1);
  uint32_t y2t[FEW_ROWS ? NF : 1][NR];
  float acc1[NF][NU][4], acc2[FEW_ROWS ? 1 : NF][NU][4];
#pragma unroll
  for (int i = 0; i < NF; ++i) {
    if constexpr (FEW_ROWS) {
#pragma unroll
      for (int c = 0; c < NR; ++c) y2t[i][c] = movm(y2[i][c]);
    }
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        acc1[i][u][e] = 0.f;
        if constexpr (!FEW_ROWS) acc2[i][u][e] = 0.f;
      }
  }

  for (int i0 = begin; i0 < end; i0 += 16) {
    float p[NF][4], ds[NF][4];
#pragma unroll
    for (int i = 0; i < NF; ++i) {
      float s[4] = {0.f, 0.f, 0.f, 0.f};
      ds[i][0] = ds[i][1] = ds[i][2] = ds[i][3] = 0.f;
#pragma unroll
      for (int c = 0; c < NR; c += 2) {
        Mma<T>::run(s, x1[0][c], x1[1][c], x1[0][c + 1], x1[1][c + 1], y1[i][c], y1[i][c + 1]);
        Mma<T>::run(ds[i], x2[0][c], x2[1][c], x2[0][c + 1], x2[1][c + 1], y2[i][c], y2[i][c + 1]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[i][e] = fmaf(s[e], a.c, FEW_ROWS ? xs[e >> 1] : fs[i][e & 1]);
        if constexpr (FEW_ROWS) p[i][e] = ex2f(p[i][e] - fs[i][e & 1]);
      }
    }
    if constexpr (!FEW_ROWS) {
      // all keys are here: the whole softmax and D from these logits and dp themselves, so that a query with
      // one key has p = 1 and dS = 0 exactly, and the forward pass leaves nothing but its inputs
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float m = kXmNone, l = 0.f, f = 0.f;
#pragma unroll
        for (int i = 0; i < NF; ++i) m = fmaxf(m, fmaxf(p[i][2 * h], p[i][2 * h + 1]));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
#pragma unroll
        for (int i = 0; i < NF; ++i) {
          p[i][2 * h] = ex2f(p[i][2 * h] - m), p[i][2 * h + 1] = ex2f(p[i][2 * h + 1] - m);
          l += p[i][2 * h] + p[i][2 * h + 1];
        }
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        l = l == 0.f ? 0.f : rcp_fast(l);
#pragma unroll
        for (int i = 0; i < NF; ++i) {
          p[i][2 * h] *= l, p[i][2 * h + 1] *= l;
          f = fmaf(p[i][2 * h], ds[i][2 * h], fmaf(p[i][2 * h + 1], ds[i][2 * h + 1], f));
        }
        f += __shfl_xor_sync(0xffffffffu, f, 1);
        xd[h] = f + __shfl_xor_sync(0xffffffffu, f, 2);
      }
    }
    Turned<T, 2, NR> x1t;
    x1t.make(x1);
    uint32_t x2t[2][FEW_ROWS ? 1 : NR];
    if constexpr (!FEW_ROWS) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < NR; ++c) x2t[h][c] = movm(x2[h][c]);
    }
    // keys that are not there leave zeros, also where a query or its gradient is not finite
    const bool gone[2] = {FEW_ROWS && xs[0] != 0.f, FEW_ROWS && xs[1] != 0.f};
    if (i0 + 16 < end) load_long(i0 + 16);   // the next step's, under this one's arithmetic
    float e1[NR][4], e2[FEW_ROWS ? NR : 1][4];
#pragma unroll
    for (int c = 0; c < NR; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        e1[c][e] = 0.f;
        if constexpr (FEW_ROWS) e2[c][e] = 0.f;
      }
    constexpr int PAIR = NF > 1 ? 2 : 1;
#pragma unroll
    for (int i = 0; i < NF; i += PAIR) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int x = 0; x < PAIR; ++x) {
#pragma unroll
        for (int e = 0; e < 4; ++e) ds[i + x][e] = p[i + x][e] * (ds[i + x][e] - (FEW_ROWS ? fd[i + x][e & 1] : xd[e >> 1]));
        split2<__nv_bfloat16>(ds[i + x][0], ds[i + x][1], hi[2 * x], lo[2 * x]);
        split2<__nv_bfloat16>(ds[i + x][2], ds[i + x][3], hi[2 * x + 1], lo[2 * x + 1]);
        const uint32_t h0 = movm(hi[2 * x]), h1 = movm(hi[2 * x + 1]), l0 = movm(lo[2 * x]), l1 = movm(lo[2 * x + 1]);
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          float(&c)[4] = acc1[i + x][u];
          B16::run(c, x1t.hi[0][2 * u], x1t.hi[0][2 * u + 1], x1t.hi[1][2 * u], x1t.hi[1][2 * u + 1], h0, h1);
          B16::run(c, x1t.hi[0][2 * u], x1t.hi[0][2 * u + 1], x1t.hi[1][2 * u], x1t.hi[1][2 * u + 1], l0, l1);
          if constexpr (kIsHalf<T>)
            B16::run(c, x1t.lo[0][2 * u], x1t.lo[0][2 * u + 1], x1t.lo[1][2 * u], x1t.lo[1][2 * u + 1], h0, h1);
        }
      }
      if constexpr (PAIR == 2) {
        ds_product<T, NF, NR>(e1, hi, lo, y1t, i);
      } else {
#pragma unroll
        for (int c = 0; c < NR; ++c) {
          B16::run8(e1[c], hi[0], hi[1], y1t.hi[0][c]);
          B16::run8(e1[c], lo[0], lo[1], y1t.hi[0][c]);
          if constexpr (kIsHalf<T>) B16::run8(e1[c], hi[0], hi[1], y1t.lo[0][c]);
        }
      }
#pragma unroll
      for (int x = 0; x < PAIR; ++x) {
        p_terms<T>(p[i + x][0] * kP, p[i + x][1] * kP, hi[2 * x], lo[2 * x]);
        p_terms<T>(p[i + x][2] * kP, p[i + x][3] * kP, hi[2 * x + 1], lo[2 * x + 1]);
        if constexpr (!FEW_ROWS) {
          const uint32_t h0 = movm(hi[2 * x]), h1 = movm(hi[2 * x + 1]), l0 = movm(lo[2 * x]), l1 = movm(lo[2 * x + 1]);
#pragma unroll
          for (int u = 0; u < NU; ++u) {
            float(&c)[4] = acc2[i + x][u];
            if constexpr (kIsHalf<T>) {
              float rest[4] = {0.f, 0.f, 0.f, 0.f};
              Mma<T>::run(rest, x2t[0][2 * u], x2t[0][2 * u + 1], x2t[1][2 * u], x2t[1][2 * u + 1], l0, l1);
#pragma unroll
              for (int e = 0; e < 4; ++e) c[e] = fmaf(rest[e], 1.f / 2048.f, c[e]);
            } else {
              Mma<T>::run(c, x2t[0][2 * u], x2t[0][2 * u + 1], x2t[1][2 * u], x2t[1][2 * u + 1], l0, l1);
            }
            Mma<T>::run(c, x2t[0][2 * u], x2t[0][2 * u + 1], x2t[1][2 * u], x2t[1][2 * u + 1], h0, h1);
          }
        }
      }
      if constexpr (FEW_ROWS) {
#pragma unroll
        for (int c = 0; c < NR; ++c) {
          float rest[4] = {0.f, 0.f, 0.f, 0.f};
          float(&low)[4] = kIsHalf<T> ? rest : e2[c];
          if constexpr (PAIR == 2) {
            Mma<T>::run(low, lo[0], lo[1], lo[2], lo[3], y2t[i][c], y2t[i + 1][c]);
            Mma<T>::run(e2[c], hi[0], hi[1], hi[2], hi[3], y2t[i][c], y2t[i + 1][c]);
          } else {
            Mma<T>::run8(low, lo[0], lo[1], y2t[0][c]);
            Mma<T>::run8(e2[c], hi[0], hi[1], y2t[0][c]);
          }
          if constexpr (kIsHalf<T>) {
#pragma unroll
            for (int e = 0; e < 4; ++e) e2[c][e] = fmaf(rest[e], 1.f / 2048.f, e2[c][e]);
          }
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = i0 + h * 8 + g;
      if (i >= end) continue;
      uint32_t y[NR];
#pragma unroll
      for (int c = 0; c < NR; ++c) y[c] = gone[h] ? 0u : Mma<T>::pack(e1[c][2 * h] * a.scale, e1[c][2 * h + 1] * a.scale);
      if constexpr (FEW_ROWS) {
        if (a.dk != nullptr) {
          const int64_t to = ((static_cast<int64_t>(b) * a.Tk + i) * a.kv_heads + n) * a.d;
          store_frag<T, DP>(static_cast<T*>(a.dk) + to, t, a.d, y);
#pragma unroll
          for (int c = 0; c < NR; ++c) y[c] = gone[h] ? 0u : Mma<T>::pack(e2[c][2 * h] * (1.f / kP), e2[c][2 * h + 1] * (1.f / kP));
          store_frag<T, DP>(static_cast<T*>(a.dv) + to, t, a.d, y);
        }
      } else if (a.dq != nullptr) {
        store_frag<T, DP>(static_cast<T*>(a.dq) + row_dense(a, b, n, i), t, a.d, y);
      }
    }
  }

  if constexpr (FEW_ROWS) {
    if (!__any_sync(0xffffffffu, some)) {    // as in the forward pass
#pragma unroll
      for (int i = 0; i < NF; ++i)
#pragma unroll
        for (int u = 0; u < NU; ++u) acc1[i][u][0] = acc1[i][u][1] = acc1[i][u][2] = acc1[i][u][3] = 0.f;
    }
  }

  // join the few side's sums of the warps and the cluster, in a fixed order
  constexpr int N1 = NF * NU * 4, NREG = FEW_ROWS ? N1 : 2 * N1;   // [8][NREG][32]; the block's sums end up in [0]
#pragma unroll
  for (int w = 0; w < N1; ++w) {
    xsm[(warp * NREG + w) * 32 + lane] = acc1[w / 4 / NU][w / 4 % NU][w % 4];
    if constexpr (!FEW_ROWS) xsm[(warp * NREG + N1 + w) * 32 + lane] = acc2[w / 4 / NU][w / 4 % NU][w % 4];
  }
  __syncthreads();
  for (int w = warp; w < NREG; w += kXmWarps) {
    float x = 0.f;
#pragma unroll
    for (int z = 0; z < kXmWarps; ++z) x += xsm[(z * NREG + w) * 32 + lane];
    xsm[w * 32 + lane] = x;                                        // read by this lane only so far
  }
  if (cl > 1) cluster_sync_all(); else __syncthreads();
  const uint32_t base = smem_u32(xsm) + lane * 4;
  for (int w = rank * kXmWarps + warp; w < NREG; w += cl * kXmWarps) {
    const bool second = w >= N1;
    const int v = second ? w - N1 : w, e = v % 4, u = v / 4 % NU, f = v / 4 / NU * 8 + 2 * t + (e & 1);
    float x = 0.f;
    for (int z = 0; z < cl; ++z) x += ld_dsmem(mapa_shared(base, z) + w * 128);
    if (!FEW_ROWS && !key_ok(f)) x = 0.f;
    const int ch = g / 2 * (DP / 4) + 4 * u + g % 2 + (e & 2);
    T* to = static_cast<T*>(FEW_ROWS ? a.dq : second ? a.dv : a.dk);
    if (f < (FEW_ROWS ? rows : a.Tk) && ch < a.d && to != nullptr) {
      const int64_t at = FEW_ROWS ? row_dense(a, b, n, f) : ((static_cast<int64_t>(b) * a.Tk + f) * a.kv_heads + n) * a.d;
      store1(to + at + ch, x * (second ? 1.f / kP : a.scale));
    }
  }
  if (cl > 1) cluster_sync_all();
}

// ---------------------------------------------------------------------------
// Launch rules
// ---------------------------------------------------------------------------
// Blocks per cluster: blocks are added along the long side until every SM has one, while each warp
// keeps at least one step. (Two per SM measured slower: 64 pairs of 4096 keys forward 17 us against 12,
// the join outweighs the shorter walks.)
static int xattn_cluster(int64_t blocks, int other, int step, int most = 8) {
  int c = 1;
  // 16 only where the warps of 8 blocks would walk four steps or more (4096 keys: 4.95 us with 8, 5.4 with 16;
  // 16384 keys: 8.8 and 7.4)
  while (c < most && (c < 8 || (blocks * 16 <= 148 && other >= 32 * kXmWarps * step)) && blocks * c < 148 && other > c * kXmWarps * step) c *= 2;
  return c;
}
template <class T, int DP, int NQ, int HP = 1>
static int xattn_few_rows_launch(const XAttn& a, cudaStream_t stream) {
  const int rows = a.group * a.Tq, tiles = (rows + 8 * NQ - 1) / (8 * NQ);
  constexpr size_t smem = (kXmWarps * HP * 8 * NQ + HP * 8 * NQ + kXmWarps * NQ * (DP / 4 + 2) * 32) * sizeof(float);
  static PerDeviceOnce once;
  static ClusterLimit limit;
  const int st = allow_smem(once, xattn_fwd_few_rows<T, DP, NQ, HP>, smem);
  if (st != SSAM_OK) return st;
  const int cl = xattn_cluster(static_cast<int64_t>(a.B) * (a.kv_heads / HP) * tiles, a.Tk, DP <= 32 ? 32 : 16,
                               limit.get(xattn_fwd_few_rows<T, DP, NQ, HP>, kXmThreads, smem));
  return launch_following(xattn_fwd_few_rows<T, DP, NQ, HP>, dim3(tiles * cl, a.kv_heads / HP, a.B), kXmThreads, smem, cl,
                        stream, a, 0);
}

template <class T, int DP, int NK, int HP = 1>
static int xattn_few_keys_launch(const XAttn& a, cudaStream_t stream) {
  const int tiles = (a.Tq + 15) / 16;
  const int64_t pairs = static_cast<int64_t>(a.B) * (a.heads / HP);
  // row shares: at least 4 tiles each (the K, V fragments are loaded once per share), about 64 warps per SM
  const int64_t want = (148 * 64 + pairs - 1) / pairs;
  const int chunks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want, (tiles + 3) / 4)));
  const int64_t blocks = (pairs * chunks + kXmWarps - 1) / kXmWarps;
  return launch_following(xattn_fwd_few_keys<T, DP, NK, HP>, dim3(static_cast<unsigned>(blocks)), kXmThreads, 0, 1, stream,
                        a, chunks);
}

// Heads of 16 that lie side by side in every tensor can be read two at a time.
static bool xattn_paired(const XAttn& a) {
  return a.d == 16 && a.group == 1 && a.heads % 2 == 0 && a.qs[2] == 16 && a.ks[2] == 16 && a.vs[2] == 16 && a.os[2] == 16;
}

template <class T, int DP, int NF, bool FEW_ROWS>
static int xattn_bwd_few_launch(const XAttn& a, cudaStream_t stream) {
  constexpr size_t smem = kXmWarps * (FEW_ROWS ? 1 : 2) * NF * (DP / 4) * 32 * sizeof(float);
  static PerDeviceOnce once;
  static ClusterLimit limit;
  const int st = allow_smem(once, xattn_bwd_few<T, DP, NF, FEW_ROWS>, smem);
  if (st != SSAM_OK) return st;
  const int cl = xattn_cluster(static_cast<int64_t>(a.B) * a.kv_heads, FEW_ROWS ? a.Tk : a.group * a.Tq, 16,
                               limit.get(xattn_bwd_few<T, DP, NF, FEW_ROWS>, kXmThreads, smem));
  return launch_following(xattn_bwd_few<T, DP, NF, FEW_ROWS>, dim3(cl, a.kv_heads, a.B), kXmThreads, smem, cl, stream, a,
                        0);
}
// the smallest instance that holds `few` entries
template <class T, int DP, bool FEW_ROWS>
static int xattn_bwd_few_pick(const XAttn& a, int few, cudaStream_t stream) {
  if constexpr (kXmFewTiles<DP> >= 8) {
    if (few > 32) return xattn_bwd_few_launch<T, DP, 8, FEW_ROWS>(a, stream);
  }
  if constexpr (kXmFewTiles<DP> >= 4) {
    if (few > 16) return xattn_bwd_few_launch<T, DP, 4, FEW_ROWS>(a, stream);
  }
  if constexpr (kXmFewTiles<DP> >= 2) {
    if (few > 8) return xattn_bwd_few_launch<T, DP, 2, FEW_ROWS>(a, stream);
  }
  return xattn_bwd_few_launch<T, DP, 1, FEW_ROWS>(a, stream);
}

template <class T, int DP>
static int xattn_mma_dp(const XAttn& a, bool backward, cudaStream_t stream) {
  const int rows = a.group * a.Tq;
  if (!backward) {
    if constexpr (DP == 16) {
      // two heads to a warp where that leaves every SM a block (and every row 16-byte pieces)
      if (xattn_paired(a)) {
        const int64_t pairs = static_cast<int64_t>(a.B) * a.heads;
        if (a.Tk <= 8) return xattn_few_keys_launch<T, 32, 1, 2>(a, stream);
        if (a.Tk <= 16) return xattn_few_keys_launch<T, 32, 2, 2>(a, stream);
        if (a.Tk > 64 && pairs >= 2 * 148 && rows <= 8) return xattn_few_rows_launch<T, 32, 1, 2>(a, stream);
        if (a.Tk > 64 && pairs >= 2 * 148 && rows <= 16) return xattn_few_rows_launch<T, 32, 2, 2>(a, stream);
      }
    }
    if (a.Tk <= 8) return xattn_few_keys_launch<T, DP, 1>(a, stream);
    if (a.Tk <= 16) return xattn_few_keys_launch<T, DP, 2>(a, stream);
    if constexpr (kXmKeyTiles<DP> >= 4) {
      if (a.Tk <= 32) return xattn_few_keys_launch<T, DP, 4>(a, stream);
    }
    if constexpr (kXmKeyTiles<DP> >= 8) {
      if (a.Tk <= 64) return xattn_few_keys_launch<T, DP, 8>(a, stream);
    }
    if (rows <= 8) return xattn_few_rows_launch<T, DP, 1>(a, stream);
    if (rows <= 16) return xattn_few_rows_launch<T, DP, 2>(a, stream);
    if constexpr (kXmRowTiles<DP> >= 4) {        // up to 32 rows to a block: two blocks of 24 or 32 past that
      if (rows <= 24 || (rows > 32 && rows <= 48 && kXmRowTiles<DP> == 8)) return xattn_few_rows_launch<T, DP, 3>(a, stream);
      if (rows <= 8 * kXmRowTiles<DP>) return xattn_few_rows_launch<T, DP, 4>(a, stream);
    }
    return xattn_tc(a, kIsHalf<T> ? 0 : 1, false, stream);
  }
  if (a.Tk <= 8 * kXmFewTiles<DP>) return xattn_bwd_few_pick<T, DP, false>(a, a.Tk, stream);
  if (rows <= 8 * kXmFewTiles<DP>) return xattn_bwd_few_pick<T, DP, true>(a, rows, stream);
  return xattn_tc(a, kIsHalf<T> ? 0 : 1, true, stream);
}

template <class T>
static int xattn_mma(const XAttn& a, bool backward, cudaStream_t stream) {
  if (a.d <= 16) return xattn_mma_dp<T, 16>(a, backward, stream);
  if (a.d <= 32) return xattn_mma_dp<T, 32>(a, backward, stream);
  if (a.d <= 64) return xattn_mma_dp<T, 64>(a, backward, stream);
  return xattn_mma_dp<T, 128>(a, backward, stream);
}

}  // namespace ssam
