// Tensor-core kernels of the cross attention for fp16 / bf16 (included by
// cross_attention.cu, which has the formulas and the conventions).
//
// Everything is built from mma.m16n8k16 on registers: head sizes here are 16 to 128
// and one of the two token sets is usually a handful of prompt tokens, so a warp's
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
#pragma once

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
  static __device__ __forceinline__ uint32_t pack(float x, float y) { return pack_bf16x2(x, y); }
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
};

__device__ __forceinline__ uint32_t movm(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// x, y -> packed value and packed remainder
template <class T>
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = Mma<T>::pack(x, y);
  const float2 h = Mma<T>::unpack(hi);
  lo = Mma<T>::pack(x - h.x, y - h.y);
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

// Sums acc over the block's warps into warp 0 (pairwise, a fixed order), through
// sm[4][NREG][32]. All threads call it.
template <int NREG>
__device__ __forceinline__ void warp_tree_sum(float* acc, float* sm, int warp, int lane) {
#pragma unroll
  for (int off = kXmWarps / 2; off >= 1; off >>= 1) {
    __syncthreads();
    if (warp >= off && warp < 2 * off) {
#pragma unroll
      for (int i = 0; i < NREG; ++i) sm[((warp - off) * NREG + i) * 32 + lane] = acc[i];
    }
    __syncthreads();
    if (warp < off) {
#pragma unroll
      for (int i = 0; i < NREG; ++i) acc[i] += sm[(warp * NREG + i) * 32 + lane];
    }
  }
}

// ---------------------------------------------------------------------------
// Forward. A warp holds 16 MT query rows of one key head and walks keys CK at a time.
// split = false: the block's 8 warps hold 8 row tiles and each walks all keys.
// split = true: one row tile per block, its keys shared by the 8 warps and the cluster.
// ---------------------------------------------------------------------------
template <class T, int DP, int MT>
__global__ void __launch_bounds__(kXmThreads) xattn_fwd_mma(const XAttn a, int split) {
  constexpr int NR = DP / 8;                 // registers of a row fragment = 8-channel blocks
  constexpr int CK = DP <= 32 ? 32 : 16;     // keys per step
  constexpr int NT = CK / 8;
  extern __shared__ __align__(16) float xsm[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int b = blockIdx.z, n = blockIdx.y;
  const int cl = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
  const int rows = a.group * a.Tq;
  const int r0 = (split ? static_cast<int>(blockIdx.x) / cl : static_cast<int>(blockIdx.x) * kXmWarps + warp) * 16 * MT;
  if (!split && r0 >= rows) return;
  const int keys = xattn_keys(a, b);
  int j_begin = 0, j_end = keys;
  if (split) {
    const int steps = (keys + CK - 1) / CK, ns = kXmWarps * cl;
    const int per = (steps + ns - 1) / ns * CK;
    j_begin = min(keys, (rank * kXmWarps + warp) * per);
    j_end = min(keys, j_begin + per);
  }
  const T* kb = static_cast<const T*>(a.k) + b * a.ks[0] + n * a.ks[2];
  const T* vb = static_cast<const T*>(a.v) + b * a.vs[0] + n * a.vs[2];
  const uint8_t* mask = a.key_mask == nullptr ? nullptr : a.key_mask + static_cast<int64_t>(b) * a.Tk;

  uint32_t q[MT][2][NR];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = r0 + mt * 16 + h * 8 + g;
      load_frag<T, DP>(static_cast<const T*>(a.q) + row_offset(a, a.qs, b, n, min(r, rows - 1)), t, a.d, r < rows,
                       q[mt][h]);
    }
  float o[MT][NR][4], m[MT][2], l[MT][2];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    m[mt][0] = m[mt][1] = -INFINITY, l[mt][0] = l[mt][1] = 0.f;
#pragma unroll
    for (int i = 0; i < NR; ++i) o[mt][i][0] = o[mt][i][1] = o[mt][i][2] = o[mt][i][3] = 0.f;
  }

  for (int j0 = j_begin; j0 < j_end; j0 += CK) {
    uint32_t k[NT][NR], v[NT][NR];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int j = j0 + i * 8 + g;
      const bool ok = j < j_end && (mask == nullptr || __ldg(mask + j) != 0);
      load_frag<T, DP>(kb + j * a.ks[1], t, a.d, ok, k[i]);
      load_frag<T, DP>(vb + j * a.vs[1], t, a.d, ok, v[i]);
    }
    const bool edge = j0 + CK > j_end || mask != nullptr;
    uint32_t there = 0xffffffffu;            // bit 2i + e: key j0 + 8i + 2t + e
    if (edge) {
      there = 0;
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = j0 + i * 8 + 2 * t + e;
          if (j < j_end && (mask == nullptr || __ldg(mask + j) != 0)) there |= 1u << (2 * i + e);
        }
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int c = 0; c < NR; ++c) v[i][c] = movm(v[i][c]);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float s[NT][4];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
        for (int c = 0; c < NR; c += 2)
          Mma<T>::run(s[i], q[mt][0][c], q[mt][1][c], q[mt][0][c + 1], q[mt][1][c + 1], k[i][c], k[i][c + 1]);
      }
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[i][e] = __fmul_rn(s[i][e], a.c);
          if (edge && !(there >> (2 * i + (e & 1)) & 1u)) s[i][e] = -INFINITY;
          mx[e >> 1] = fmaxf(mx[e >> 1], s[i][e]);
        }
      float use[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
        mx[h] = fmaxf(mx[h], m[mt][h]);
        use[h] = mx[h] == -INFINITY ? 0.f : mx[h];   // no key so far: 2^(-inf - 0) = 0
        const float f = ex2f(m[mt][h] - use[h]);
        m[mt][h] = mx[h];
        l[mt][h] *= f;
#pragma unroll
        for (int c = 0; c < NR; ++c) o[mt][c][2 * h] *= f, o[mt][c][2 * h + 1] *= f;
      }
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[i][e] = ex2f(__fsub_rn(s[i][e], use[e >> 1]));
          l[mt][e >> 1] += s[i][e];
        }
#pragma unroll
      for (int i = 0; i < NT; i += 2) {
        uint32_t hi[4], lo[4];
        split2<T>(s[i][0], s[i][1], hi[0], lo[0]);
        split2<T>(s[i][2], s[i][3], hi[1], lo[1]);
        split2<T>(s[i + 1][0], s[i + 1][1], hi[2], lo[2]);
        split2<T>(s[i + 1][2], s[i + 1][3], hi[3], lo[3]);
#pragma unroll
        for (int c = 0; c < NR; ++c) {
          Mma<T>::run(o[mt][c], hi[0], hi[1], hi[2], hi[3], v[i][c], v[i + 1][c]);
          Mma<T>::run(o[mt][c], lo[0], lo[1], lo[2], lo[3], v[i][c], v[i + 1][c]);
        }
      }
    }
  }

  // the lanes of a quad share a row
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[mt][h] += __shfl_xor_sync(0xffffffffu, l[mt][h], 1);
      l[mt][h] += __shfl_xor_sync(0xffffffffu, l[mt][h], 2);
    }
  const int64_t stat0 = (static_cast<int64_t>(b) * a.heads + n * a.group) * a.Tq;
  if (!split) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = r0 + mt * 16 + h * 8 + g;
        if (r >= rows) continue;
        const float inv = l[mt][h] == 0.f ? 0.f : 1.f / l[mt][h];
        uint32_t y[NR];
#pragma unroll
        for (int c = 0; c < NR; ++c) y[c] = Mma<T>::pack(o[mt][c][2 * h] * inv, o[mt][c][2 * h + 1] * inv);
        store_frag<T, DP>(static_cast<T*>(a.out) + row_offset(a, a.os, b, n, r), t, a.d, y);
        if (a.lse != nullptr && t == 0) a.lse[stat0 + r] = l[mt][h] == 0.f ? INFINITY : m[mt][h] + log2f(l[mt][h]);
        if (a.out_f32 != nullptr) {
          float* f = a.out_f32 + row_dense(a, b, n, r) + t * (DP / 4);
#pragma unroll
          for (int c = 0; c < NR; ++c)
            if (t * (DP / 4) + 2 * c < a.d)
              *reinterpret_cast<float2*>(f + 2 * c) = make_float2(o[mt][c][2 * h] * inv, o[mt][c][2 * h + 1] * inv);
        }
      }
    return;
  }
  // Join: the common maximum of the block's warps, then of the cluster's blocks; every warp
  // rescales its share to it, the shares are summed, and the sums divided on the way out.
  constexpr int NREG = MT * (NR * 4 + 2), ROWS = 16 * MT;
  float* s_top = xsm;                        // [8][ROWS]
  float* s_acc = xsm + kXmWarps * ROWS;      // [4][NREG][32]
  float acc[NREG];
  if (t == 0) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) s_top[warp * ROWS + mt * 16 + h * 8 + g] = m[mt][h];
  }
  __syncthreads();
  float top[MT][2];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float x = -INFINITY;
#pragma unroll
      for (int w = 0; w < kXmWarps; ++w) x = fmaxf(x, s_top[w * ROWS + mt * 16 + h * 8 + g]);
      top[mt][h] = x;
    }
  if (cl > 1) {
    __syncthreads();
    if (warp == 0 && t == 0) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) s_top[mt * 16 + h * 8 + g] = top[mt][h];
    }
    cluster_sync_all();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t at = smem_u32(s_top + mt * 16 + h * 8 + g);
        for (int i = 0; i < cl; ++i) top[mt][h] = fmaxf(top[mt][h], ld_dsmem(mapa_shared(at, i)));
      }
  }
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float f = m[mt][h] == -INFINITY && !(l[mt][h] != l[mt][h]) ? 0.f : ex2f(m[mt][h] - top[mt][h]);
      acc[mt * (NR * 4 + 2) + NR * 4 + h] = l[mt][h] * f;
#pragma unroll
      for (int c = 0; c < NR; ++c) {
        acc[mt * (NR * 4 + 2) + c * 4 + 2 * h] = o[mt][c][2 * h] * f;
        acc[mt * (NR * 4 + 2) + c * 4 + 2 * h + 1] = o[mt][c][2 * h + 1] * f;
      }
    }
  warp_tree_sum<NREG>(acc, s_acc, warp, lane);
  __syncthreads();
  if (warp == 0) {
#pragma unroll
    for (int i = 0; i < NREG; ++i) s_acc[i * 32 + lane] = acc[i];
  }
  if (cl > 1) cluster_sync_all(); else __syncthreads();
  const uint32_t base = smem_u32(s_acc) + lane * 4;
  for (int u = rank * kXmWarps + warp; u < MT * 2 * NR; u += cl * kXmWarps) {
    const int mt = u / (2 * NR), h = u / NR % 2, c = u % NR;
    const int ro = mt * 16 + h * 8 + g, r = r0 + ro;
    const int i0 = mt * (NR * 4 + 2) + c * 4 + 2 * h, il = mt * (NR * 4 + 2) + NR * 4 + h;
    float x = 0.f, y = 0.f, den = 0.f, mm = -INFINITY;
    for (int i = 0; i < cl; ++i) {
      const uint32_t from = mapa_shared(base, i);
      x += ld_dsmem(from + i0 * 128);
      y += ld_dsmem(from + (i0 + 1) * 128);
      den += ld_dsmem(from + il * 128);
      if (cl > 1) mm = fmaxf(mm, ld_dsmem(mapa_shared(smem_u32(s_top + ro), i)));
    }
    if (cl == 1) mm = -INFINITY;
    if (r < rows) {
      const float inv = den == 0.f ? 0.f : 1.f / den;
      const int ch = t * (DP / 4) + 2 * c;
      if (ch < a.d) {
        *reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + row_offset(a, a.os, b, n, r) + ch) =
            Mma<T>::pack(x * inv, y * inv);
        if (a.out_f32 != nullptr)
          *reinterpret_cast<float2*>(a.out_f32 + row_dense(a, b, n, r) + ch) = make_float2(x * inv, y * inv);
      }
      if (a.lse != nullptr && c == 0 && t == 0) {
        if (cl == 1)
          for (int w = 0; w < kXmWarps; ++w) mm = fmaxf(mm, s_top[w * ROWS + ro]);
        a.lse[stat0 + r] = den == 0.f ? INFINITY : mm + log2f(den);
      }
    }
  }
  if (cl > 1) cluster_sync_all();
}

// ---------------------------------------------------------------------------
// Backward. A warp owns 16 M entries of one token set (OWN_ROWS: query rows, with
// x1 = q, x2 = dout; else keys, with x1 = k, x2 = v) and walks the other set
// 16 entries at a time (y1 = k or q, y2 = v or dout):
//   s = x1 y1^T, dp = x2 y2^T, p = 2^(c s - lse), ds = p (dp - D)      (own x other)
//   own rows:  dq += ds k              own keys:  dk += ds q,  dv += p dout
// FUSED: the owned entries are all there are on that side, so the other side's
// gradients of a step are complete as well and leave at once, from the turned blocks:
//   own rows:  dk = ds^T q, dv = p^T dout        own keys:  dq = ds^T k
// Owned sums of the block's 8 warps and the cluster are joined at the end.
//
// fp16: dS has no fixed scale (it follows the loss), so its products run in bf16, which
// has fp32's range: dS as two bf16 terms, the fp16 factor as two bf16 terms (exact,
// 11 = 8 + 3 bits), without the product of the two remainders. P lies in [0, 1] and
// is scaled by 2^12, so that its fp16 remainder keeps digits down to 2^-36.
// ---------------------------------------------------------------------------
template <class T>
constexpr bool kIsHalf = false;
template <>
constexpr bool kIsHalf<__half> = true;

// B operand (tokens as k) of one 16-token tile: turned blocks, as bf16 for the dS products
template <class T, int NR>
struct Turned {
  uint32_t hi[2][NR], lo[2][kIsHalf<T> ? NR : 1];
  __device__ __forceinline__ void make(const uint32_t (&x)[2][NR]) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
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
template <class T, int NR>
__device__ __forceinline__ void ds_product(float (&acc)[NR][4], const uint32_t (&hi)[4], const uint32_t (&lo)[4],
                                           const Turned<T, NR>& y) {
  using B = Mma<__nv_bfloat16>;
#pragma unroll
  for (int c = 0; c < NR; ++c) {
    B::run(acc[c], hi[0], hi[1], hi[2], hi[3], y.hi[0][c], y.hi[1][c]);
    B::run(acc[c], lo[0], lo[1], lo[2], lo[3], y.hi[0][c], y.hi[1][c]);
    if constexpr (kIsHalf<T>) B::run(acc[c], hi[0], hi[1], hi[2], hi[3], y.lo[0][c], y.lo[1][c]);
  }
}

template <class T, int DP, int M, bool OWN_ROWS, bool FUSED>
__global__ void __launch_bounds__(kXmThreads) xattn_bwd_mma(const XAttn a, int) {
  constexpr int NR = DP / 8;
  constexpr float kP = kIsHalf<T> ? 4096.f : 1.f;
  extern __shared__ __align__(16) float xsm[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int b = blockIdx.z, n = blockIdx.y;
  const int cl = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
  const int rows = a.group * a.Tq, keys = xattn_keys(a, b);
  const int own0 = static_cast<int>(blockIdx.x) / cl * 16 * M;
  const T* qb = static_cast<const T*>(a.q);
  const T* ob = static_cast<const T*>(a.dout);
  const T* kb = static_cast<const T*>(a.k) + b * a.ks[0] + n * a.ks[2];
  const T* vb = static_cast<const T*>(a.v) + b * a.vs[0] + n * a.vs[2];
  const uint8_t* mask = a.key_mask == nullptr ? nullptr : a.key_mask + static_cast<int64_t>(b) * a.Tk;
  const int64_t stat0 = (static_cast<int64_t>(b) * a.heads + n * a.group) * a.Tq;
  auto key_ok = [&](int j) { return j < keys && (mask == nullptr || __ldg(mask + j) != 0); };
  auto load_row = [&](int r, uint32_t(&x1)[NR], uint32_t(&x2)[NR]) {
    const int rr = min(r, rows - 1);
    load_frag<T, DP>(qb + row_offset(a, a.qs, b, n, rr), t, a.d, r < rows, x1);
    load_frag<T, DP>(ob + row_offset(a, a.os, b, n, rr), t, a.d, r < rows, x2);
  };
  auto load_key = [&](int j, uint32_t(&x1)[NR], uint32_t(&x2)[NR]) {
    const bool ok = key_ok(j);
    load_frag<T, DP>(kb + j * a.ks[1], t, a.d, ok, x1);
    load_frag<T, DP>(vb + j * a.vs[1], t, a.d, ok, x2);
  };

  uint32_t x1[M][2][NR], x2[M][2][NR];
  float lse_own[M][2], delta_own[M][2];      // own rows
  bool ok_own[M][2];                         // own keys
#pragma unroll
  for (int mt = 0; mt < M; ++mt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = own0 + mt * 16 + h * 8 + g;
      if constexpr (OWN_ROWS) {
        load_row(i, x1[mt][h], x2[mt][h]);
        lse_own[mt][h] = i < rows ? __ldg(a.lse + stat0 + i) : INFINITY;
        float f = 0.f;
        if (i < rows) {
          const float* o32 = a.out_f32 + row_dense(a, b, n, i) + t * (DP / 4);
#pragma unroll
          for (int c = 0; c < NR; ++c) {
            if (t * (DP / 4) + 2 * c >= a.d) break;
            const float2 o = __ldg(reinterpret_cast<const float2*>(o32 + 2 * c)), x = Mma<T>::unpack(x2[mt][h][c]);
            f = fmaf(o.x, x.x, f);
            f = fmaf(o.y, x.y, f);
          }
        }
        f += __shfl_xor_sync(0xffffffffu, f, 1);
        f += __shfl_xor_sync(0xffffffffu, f, 2);
        delta_own[mt][h] = f;
        if (!FUSED && rank == 0 && warp == 0 && t == 0 && i < rows) a.delta[stat0 + i] = f;
      } else {
        load_key(i, x1[mt][h], x2[mt][h]);
        ok_own[mt][h] = key_ok(i);
      }
    }
  if (OWN_ROWS && !FUSED && a.dq == nullptr) return;

  float acc1[M][NR][4];                                // dq or dk
  float acc2[OWN_ROWS ? 1 : M][NR][4];                 // dv
#pragma unroll
  for (int mt = 0; mt < M; ++mt)
#pragma unroll
    for (int c = 0; c < NR; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        acc1[mt][c][e] = 0.f;
        if constexpr (!OWN_ROWS) acc2[mt][c][e] = 0.f;
      }
  Turned<T, NR> x1t[FUSED ? M : 1];
  uint32_t x2t[FUSED && OWN_ROWS ? M : 1][2][NR];
  if constexpr (FUSED) {
#pragma unroll
    for (int mt = 0; mt < M; ++mt) {
      x1t[mt].make(x1[mt]);
      if constexpr (OWN_ROWS) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int c = 0; c < NR; ++c) x2t[mt][h][c] = movm(x2[mt][h][c]);
      }
    }
  }

  // own rows, fused: the zero gradients of the keys behind keys are written too
  const int total = OWN_ROWS ? (FUSED ? a.Tk : keys) : (FUSED || own0 < keys ? rows : 0);
  const int steps = (total + 15) / 16, ns = kXmWarps * cl;
  const int per = (steps + ns - 1) / ns * 16;
  const int begin = min(total, (rank * kXmWarps + warp) * per), end = min(total, begin + per);
  for (int i0 = begin; i0 < end; i0 += 16) {
    uint32_t y1[2][NR], y2[2][NR];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (OWN_ROWS)
        load_key(i0 + h * 8 + g, y1[h], y2[h]);
      else
        load_row(i0 + h * 8 + g, y1[h], y2[h]);
    }
    float lse[2][2], delta[2][2];            // of other entries i0 + 8 nt + 2t + e (own keys)
    bool ok[2][2];                           // (own rows)
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = i0 + nt * 8 + 2 * t + e;
        if constexpr (OWN_ROWS) {
          ok[nt][e] = key_ok(i);
        } else {
          lse[nt][e] = i < rows ? __ldg(a.lse + stat0 + i) : INFINITY;
          delta[nt][e] = FUSED || i >= rows ? 0.f : __ldg(a.delta + stat0 + i);
        }
      }
    Turned<T, NR> y1t;
    uint32_t y2t[OWN_ROWS ? 1 : 2][NR];
    y1t.make(y1);
    if constexpr (!OWN_ROWS) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < NR; ++c) y2t[h][c] = movm(y2[h][c]);
    }
    float p[M][2][4], dp[M][2][4];
#pragma unroll
    for (int mt = 0; mt < M; ++mt)
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        dp[mt][nt][0] = dp[mt][nt][1] = dp[mt][nt][2] = dp[mt][nt][3] = 0.f;
#pragma unroll
        for (int c = 0; c < NR; c += 2) {
          Mma<T>::run(s, x1[mt][0][c], x1[mt][1][c], x1[mt][0][c + 1], x1[mt][1][c + 1], y1[nt][c], y1[nt][c + 1]);
          Mma<T>::run(dp[mt][nt], x2[mt][0][c], x2[mt][1][c], x2[mt][0][c + 1], x2[mt][1][c + 1], y2[nt][c],
                      y2[nt][c + 1]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool valid = OWN_ROWS ? ok[nt][e & 1] : ok_own[mt][e >> 1];
          const float st = OWN_ROWS ? lse_own[mt][e >> 1] : lse[nt][e & 1];
          p[mt][nt][e] = valid ? ex2f(__fsub_rn(__fmul_rn(s[e], a.c), st)) : 0.f;
        }
      }
    if constexpr (!OWN_ROWS && FUSED) {
      // all keys are here: D from p and dp themselves, so a query with one key has dS = 0 exactly
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float f = 0.f;
#pragma unroll
          for (int mt = 0; mt < M; ++mt) {
            f = fmaf(p[mt][nt][e], dp[mt][nt][e], f);
            f = fmaf(p[mt][nt][e + 2], dp[mt][nt][e + 2], f);
          }
          f += __shfl_xor_sync(0xffffffffu, f, 4);
          f += __shfl_xor_sync(0xffffffffu, f, 8);
          f += __shfl_xor_sync(0xffffffffu, f, 16);
          delta[nt][e] = f;
        }
    }
    float e1[FUSED ? NR : 1][4], e2[FUSED && OWN_ROWS ? NR : 1][4];   // the other side's gradients
    if constexpr (FUSED) {
#pragma unroll
      for (int c = 0; c < NR; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          e1[c][e] = 0.f;
          if constexpr (OWN_ROWS) e2[c][e] = 0.f;
        }
    }
#pragma unroll
    for (int mt = 0; mt < M; ++mt) {
      uint32_t hi[4], lo[4];
      float ds[2][4];
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float dl = OWN_ROWS ? delta_own[mt][e >> 1] : delta[nt][e & 1];
          ds[nt][e] = p[mt][nt][e] * (dp[mt][nt][e] - dl);
        }
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        split2<__nv_bfloat16>(ds[nt][0], ds[nt][1], hi[2 * nt], lo[2 * nt]);
        split2<__nv_bfloat16>(ds[nt][2], ds[nt][3], hi[2 * nt + 1], lo[2 * nt + 1]);
      }
      ds_product<T, NR>(acc1[mt], hi, lo, y1t);
      if constexpr (FUSED) {
        const uint32_t th[4] = {movm(hi[0]), movm(hi[2]), movm(hi[1]), movm(hi[3])};
        const uint32_t tl[4] = {movm(lo[0]), movm(lo[2]), movm(lo[1]), movm(lo[3])};
        ds_product<T, NR>(e1, th, tl, x1t[mt]);
      }
      if constexpr (!OWN_ROWS || FUSED) {
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          split2<T>(p[mt][nt][0] * kP, p[mt][nt][1] * kP, hi[2 * nt], lo[2 * nt]);
          split2<T>(p[mt][nt][2] * kP, p[mt][nt][3] * kP, hi[2 * nt + 1], lo[2 * nt + 1]);
        }
        if constexpr (!OWN_ROWS) {
#pragma unroll
          for (int c = 0; c < NR; ++c) {
            Mma<T>::run(acc2[mt][c], hi[0], hi[1], hi[2], hi[3], y2t[0][c], y2t[1][c]);
            Mma<T>::run(acc2[mt][c], lo[0], lo[1], lo[2], lo[3], y2t[0][c], y2t[1][c]);
          }
        } else {
          const uint32_t th[4] = {movm(hi[0]), movm(hi[2]), movm(hi[1]), movm(hi[3])};
          const uint32_t tl[4] = {movm(lo[0]), movm(lo[2]), movm(lo[1]), movm(lo[3])};
#pragma unroll
          for (int c = 0; c < NR; ++c) {
            Mma<T>::run(e2[c], th[0], th[1], th[2], th[3], x2t[mt][0][c], x2t[mt][1][c]);
            Mma<T>::run(e2[c], tl[0], tl[1], tl[2], tl[3], x2t[mt][0][c], x2t[mt][1][c]);
          }
        }
      }
    }
    if constexpr (FUSED) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int i = i0 + h * 8 + g;
        uint32_t y[NR];
#pragma unroll
        for (int c = 0; c < NR; ++c) y[c] = Mma<T>::pack(e1[c][2 * h] * a.scale, e1[c][2 * h + 1] * a.scale);
        if constexpr (OWN_ROWS) {
          if (i < a.Tk && a.dk != nullptr) {
            const int64_t to = ((static_cast<int64_t>(b) * a.Tk + i) * a.kv_heads + n) * a.d;
            store_frag<T, DP>(static_cast<T*>(a.dk) + to, t, a.d, y);
#pragma unroll
            for (int c = 0; c < NR; ++c) y[c] = Mma<T>::pack(e2[c][2 * h] * (1.f / kP), e2[c][2 * h + 1] * (1.f / kP));
            store_frag<T, DP>(static_cast<T*>(a.dv) + to, t, a.d, y);
          }
        } else if (i < rows && a.dq != nullptr) {
          store_frag<T, DP>(static_cast<T*>(a.dq) + row_dense(a, b, n, i), t, a.d, y);
        }
      }
    }
  }

  // join the owned sums of the warps and the cluster
  auto join = [&](float* acc, void* to_v, float factor, bool first) {
    constexpr int NREG = M * NR * 4;
    if (cl > 1 && !first) cluster_sync_all();          // everybody has read the previous sums
    warp_tree_sum<NREG>(acc, xsm, warp, lane);
    __syncthreads();
    if (warp == 0) {
#pragma unroll
      for (int i = 0; i < NREG; ++i) xsm[i * 32 + lane] = acc[i];
    }
    if (cl > 1) cluster_sync_all(); else __syncthreads();
    const uint32_t base = smem_u32(xsm) + lane * 4;
    for (int u = rank * kXmWarps + warp; u < M * 2 * NR; u += cl * kXmWarps) {
      const int mt = u / (2 * NR), h = u / NR % 2, c = u % NR;
      const int i = own0 + mt * 16 + h * 8 + g, i0 = (mt * NR + c) * 4 + 2 * h;
      float x = 0.f, y = 0.f;
      for (int k = 0; k < cl; ++k) {
        const uint32_t from = mapa_shared(base, k);
        x += ld_dsmem(from + i0 * 128);
        y += ld_dsmem(from + (i0 + 1) * 128);
      }
      const int ch = t * (DP / 4) + 2 * c;
      if (i < (OWN_ROWS ? rows : a.Tk) && ch < a.d && to_v != nullptr) {
        const int64_t to = OWN_ROWS ? row_dense(a, b, n, i)
                                    : ((static_cast<int64_t>(b) * a.Tk + i) * a.kv_heads + n) * a.d;
        *reinterpret_cast<uint32_t*>(static_cast<T*>(to_v) + to + ch) = Mma<T>::pack(x * factor, y * factor);
      }
    }
  };
  join(&acc1[0][0][0], OWN_ROWS ? a.dq : a.dk, a.scale, true);
  if constexpr (!OWN_ROWS) join(&acc2[0][0][0], a.dv, 1.f / kP, false);
  if (cl > 1) cluster_sync_all();
}

// ---------------------------------------------------------------------------
// Launch rules
// ---------------------------------------------------------------------------
// Owned tiles (of 16) of the fused backward kernels: what fits the register file beside
// the turned copies.
template <int DP>
constexpr int kXmFusedRows = DP == 16 ? 4 : DP == 32 ? 2 : DP == 64 ? 1 : 0;
template <int DP>
constexpr int kXmFusedKeys = DP == 16 ? 4 : DP == 32 ? 2 : DP == 64 ? 1 : 0;

// Blocks per cluster: enough blocks for two per SM, each warp with at least one step.
static int xattn_cluster(int64_t blocks, int other, int step) {
  int c = 1;
  while (c < 8 && blocks * c < 2 * 148 && other > c * kXmWarps * step) c *= 2;
  return c;
}

template <class T, int DP, int MT>
static int xattn_fwd_mma_launch(const XAttn& a, cudaStream_t stream) {
  const int rows = a.group * a.Tq, tiles = (rows + 16 * MT - 1) / (16 * MT);
  const int64_t pairs = static_cast<int64_t>(a.B) * a.kv_heads;
  constexpr int CK = DP <= 32 ? 32 : 16;
  const int64_t whole = pairs * ((tiles + kXmWarps - 1) / kXmWarps);
  if (a.Tk <= 2 * CK || whole >= 2 * 148)
    return launch_cluster(xattn_fwd_mma<T, DP, MT>, dim3((tiles + kXmWarps - 1) / kXmWarps, a.kv_heads, a.B),
                          kXmThreads, 0, 1, stream, a, 0);
  const int cl = xattn_cluster(pairs * tiles, a.Tk, CK);
  const size_t smem = (kXmWarps * 16 * MT + 4 * MT * (DP / 2 + 2) * 32) * sizeof(float);
  return launch_cluster(xattn_fwd_mma<T, DP, MT>, dim3(tiles * cl, a.kv_heads, a.B), kXmThreads, smem, cl, stream, a,
                        1);
}

template <class T, int DP, int M, bool OWN_ROWS, bool FUSED>
static int xattn_bwd_mma_launch(const XAttn& a, cudaStream_t stream) {
  const int rows = a.group * a.Tq, own = OWN_ROWS ? rows : a.Tk, other = OWN_ROWS ? a.Tk : rows;
  const int tiles = (own + 16 * M - 1) / (16 * M);
  const int cl = xattn_cluster(static_cast<int64_t>(a.B) * a.kv_heads * tiles, other, 16);
  const size_t smem = 4 * M * (DP / 2) * 32 * sizeof(float);
  return launch_cluster(xattn_bwd_mma<T, DP, M, OWN_ROWS, FUSED>, dim3(tiles * cl, a.kv_heads, a.B), kXmThreads, smem,
                        cl, stream, a, 0);
}

template <class T, int DP>
static int xattn_mma_dp(const XAttn& a, bool backward, cudaStream_t stream) {
  const int rows = a.group * a.Tq;
  if (!backward) {
    if constexpr (DP <= 64) {
      if (rows > 16) return xattn_fwd_mma_launch<T, DP, 2>(a, stream);
    }
    return xattn_fwd_mma_launch<T, DP, 1>(a, stream);
  }
  if constexpr (kXmFusedKeys<DP> >= 1) {
    if (a.Tk <= 16) return xattn_bwd_mma_launch<T, DP, 1, false, true>(a, stream);
  }
  if constexpr (kXmFusedKeys<DP> >= 2) {
    if (a.Tk <= 32) return xattn_bwd_mma_launch<T, DP, 2, false, true>(a, stream);
  }
  if constexpr (kXmFusedKeys<DP> >= 4) {
    if (a.Tk <= 64) return xattn_bwd_mma_launch<T, DP, 4, false, true>(a, stream);
  }
  if constexpr (kXmFusedRows<DP> >= 1) {
    if (rows <= 16) return xattn_bwd_mma_launch<T, DP, 1, true, true>(a, stream);
  }
  if constexpr (kXmFusedRows<DP> >= 2) {
    if (rows <= 32) return xattn_bwd_mma_launch<T, DP, 2, true, true>(a, stream);
  }
  if constexpr (kXmFusedRows<DP> >= 4) {
    if (rows <= 64) return xattn_bwd_mma_launch<T, DP, 4, true, true>(a, stream);
  }
  constexpr int M = DP <= 32 ? 2 : 1;
  const int st = xattn_bwd_mma_launch<T, DP, M, true, false>(a, stream);
  if (st != SSAM_OK || a.dk == nullptr) return st;
  return xattn_bwd_mma_launch<T, DP, M, false, false>(a, stream);
}

template <class T>
static int xattn_mma(const XAttn& a, bool backward, cudaStream_t stream) {
  if (a.d <= 16) return xattn_mma_dp<T, 16>(a, backward, stream);
  if (a.d <= 32) return xattn_mma_dp<T, 32>(a, backward, stream);
  if (a.d <= 64) return xattn_mma_dp<T, 64>(a, backward, stream);
  return xattn_mma_dp<T, 128>(a, backward, stream);
}

// Whether the backward pass reads out_f32 (else D comes from P and dP, see above).
static bool xattn_uses_out_f32(int Tk, int d, int dtype) {
  const int most = dtype == 2 ? 0 : d <= 16 ? 16 * kXmFusedKeys<16> : d <= 32 ? 16 * kXmFusedKeys<32>
                                  : d <= 64 ? 16 * kXmFusedKeys<64> : 0;
  return Tk > most;
}

}  // namespace ssam
