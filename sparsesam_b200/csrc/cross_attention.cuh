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
//
// This header: what the translation units of the operator share (cross_attention.cu: entry points and the
// fp32 kernels; cross_attention_fp16.cu, _bf16.cu: the tensor-core kernels).
#pragma once

#include <cuda_fp16.h>

#include <algorithm>

#define SSAM_NO_WAITS
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

// early where the kernels behind are small. Behind a kernel whose blocks take the whole register file (the backward pass
// with a short side), or before one, blocks that come early are packed on the first free SMs: 23 -> 27 us for a pass
// of 11 queries on 4096 keys, 18 -> 21 for 4096 on 8, fp32 49 -> 53.
__device__ __forceinline__ XAttn follow(const XAttn& args, bool early) {
  XAttn a = args;
  const int64_t zero = follow_previous(early);
  for (const void** p : {&a.q, &a.k, &a.v, &a.dout}) *p = static_cast<const char*>(*p) + zero;
  a.key_lens += zero, a.key_mask += zero, a.out_f32 += zero, a.lse += zero, a.delta += zero;
  return a;
}

// The tensor-core path (cross_attention_mma.cuh), one translation unit per type.
int xattn_fp16(const XAttn& a, bool backward, cudaStream_t stream);
int xattn_bf16(const XAttn& a, bool backward, cudaStream_t stream);

// Two long sides on the 5th-generation tensor cores (cross_attention_tc.cu): dtype 0 / 1.
int xattn_tc(const XAttn& a, int dtype, bool backward, cudaStream_t stream);

// What counts as a short side, in tiles of 8 entries that stay in registers; longer ones go to the tcgen05 kernels.
// Measured on both sides with 8 x 8 heads, 4096 entries on the long side, bf16 (mma.sync against tcgen05, us):
//   backward (with its forward), DP 16: 64 rows 56 / 93, 64 keys 59 / 118; DP 32: 32 rows 58 / 99, 32 keys 47 / 133;
//     DP 64: 16 rows 68 / 117, 16 keys 53 / 187; DP 128: 8 rows 132 / 246, 8 keys 106 / 439. The next tile spills.
//   forward, keys: DP 16: 64 keys 17.5 / 22.4; DP 32: 32 keys 12.9 / 23.4, 64 keys 31.4 / 23.8; DP 64: 32 keys
//     26.5 / 27.0; DP 128: 16 keys 40.7 / 63.9.
//   forward, rows: DP 16: 64 rows 16.5 / 29.2; DP 32: 64 rows 26.7 / 29.5; DP 64: 32 rows 29.7 / 28.7 (one batch
//     entry 17.6 / 19.4), 48 rows 41 / 29; DP 128: 16 rows 36.6 / 52.0.
template <int DP>
constexpr int kXmFewTiles = 128 / DP;
template <int DP>
constexpr int kXmKeyTiles = DP <= 16 ? 8 : DP <= 64 ? 4 : 2;
template <int DP>
constexpr int kXmRowTiles = DP <= 32 ? 8 : DP <= 64 ? 4 : 2;

// Whether the backward pass reads out_f32 and lse (else it finds them itself, see xattn_bwd_few).
inline bool xattn_uses_stats(int Tk, int d, int dtype) {
  const int few = d <= 16 ? kXmFewTiles<16> : d <= 32 ? kXmFewTiles<32> : d <= 64 ? kXmFewTiles<64> : kXmFewTiles<128>;
  return dtype == 2 || Tk > 8 * few;
}

}  // namespace ssam
