// Linear layers with 4-bit weights and group scales, bf16 activations:
//
//   y[m,n] = act(sum_g scale[n,g] sum_{k in g} x[m,k] (q[n,k] - zero[n,g]) + bias[n])
//
// Weights lie in rows of whole 128-k chunks, 64 bytes each; in a chunk word
// 4 g + c holds k = 32 c + 8 g + 0..7.  So lane group g's 16 bytes are its
// operands of four v_mfma_f32_16x16x32_bf16, each over 32 consecutive k's, and
// a group of 32 k's or more is whole products.  A word's codes (+ 8) lie in
// the nibbles 0, 4, 1, 5, ..: a shift, an AND and an OR per pair give the two
// bf16 values (16 + code + 8) / 16, exact.  The 24/16 too much (and a zero
// point) times the sum of x over the group comes off behind the products; the
// sum is one more product, with ones, in the accumulator's own layout.  The
// scale multiplies the group's fp32 result: nothing is rounded before the output.
#pragma once

#include "mfma.hpp"

namespace teeny {

struct W4Args {
  const bf16 *x;
  const int8_t *w;
  const float *scale;
  const int32_t *zero;  // or null
  const float *bias;    // or null
  bf16 *y;
  int M, N, K, groups, group, act;
  int64_t ldy;
};

// code of position j (0..7) of a word: nibble w4_nibble(j)
__host__ __device__ constexpr int w4_nibble(int j) { return (j & 1) * 4 + (j >> 1); }

__device__ __forceinline__ bf16x8 w4_values(uint32_t word) {
  u32x4 r;
  r[0] = ((word << 3) & 0x00780078u) | 0x3F803F80u;
  r[1] = ((word >> 1) & 0x00780078u) | 0x3F803F80u;
  r[2] = ((word >> 5) & 0x00780078u) | 0x3F803F80u;
  r[3] = ((word >> 9) & 0x00780078u) | 0x3F803F80u;
  return __builtin_bit_cast(bf16x8, r);
}

// Bound on few rows: reading the weights once.  A workgroup owns 16 NB output
// columns and up to 16 MB rows of x (blockIdx.y); its KW waves share out the
// chunks of K and meet in LDS in wave order.  Weights and x come straight from
// memory in their operand's layout.  SUB: groups per chunk.
template <int MB, int NB, int SUB, int KW, bool ZERO>
__global__ __launch_bounds__(64 * KW) void gemm_w4(W4Args p) {
  constexpr int LD = 16 * NB + 1;
  __shared__ float red[KW][16 * MB * LD];
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16 * NB, m0 = blockIdx.y * 16 * MB;
  const int chunks = (p.K + 127) / 128, per = (chunks + KW - 1) / KW;
  const int cb = min(chunks, w * per), ce = min(chunks, cb + per);
  const int8_t *wrow[NB];
  const float *srow[NB];
  const int32_t *zrow[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const int64_t n = min(n0 + 16 * i + r, p.N - 1);
    wrow[i] = p.w + n * chunks * 64 + 16 * g;
    srow[i] = p.scale + n * p.groups;
    zrow[i] = ZERO ? p.zero + n * p.groups : nullptr;
  }
  const bf16 *xrow[MB];
#pragma unroll
  for (int j = 0; j < MB; ++j) xrow[j] = p.x + static_cast<int64_t>(min(m0 + 16 * j + r, p.M - 1)) * p.K;

  f32x4 tot[NB][MB];
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < MB; ++j) tot[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const uint32_t one = 0x3F803F80u;
  const bf16x8 ones = __builtin_bit_cast(bf16x8, (u32x4{one, one, one, one}));
  for (int c = cb; c < ce; ++c) {
    u32x4 q[NB];
    float sc[NB][SUB];
    float zp[NB][SUB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      q[i] = *reinterpret_cast<const u32x4 *>(wrow[i] + 64 * static_cast<int64_t>(c));
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
        // groups past the last one hold no k
        const int at = min(SUB > 1 ? c * SUB + s : static_cast<int>(128 * static_cast<int64_t>(c) / p.group), p.groups - 1);
        sc[i][s] = srow[i][at];
        zp[i][s] = ZERO ? 1.5f + static_cast<float>(zrow[i][at]) * 0.0625f : 1.5f;
      }
    }
    u32x4 x[MB][4];
#pragma unroll
    for (int j = 0; j < MB; ++j)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int k = 128 * c + 32 * t + 8 * g;  // K % 8 == 0: a vector is inside or outside as a whole
        x[j][t] = *reinterpret_cast<const u32x4 *>(xrow[j] + (k < p.K ? k : 0));
        if (k >= p.K) x[j][t] = u32x4{0u, 0u, 0u, 0u};
      }
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      f32x4 acc[NB][MB], sum[MB];
#pragma unroll
      for (int j = 0; j < MB; ++j) {
        sum[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NB; ++i) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      }
#pragma unroll
      for (int t = s * 4 / SUB; t < (s + 1) * 4 / SUB; ++t) {
#pragma unroll
        for (int j = 0; j < MB; ++j)
          sum[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x[j][t]), ones, sum[j], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const bf16x8 b = w4_values(q[i][t]);
#pragma unroll
          for (int j = 0; j < MB; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x[j][t]), b, acc[i][j], 0, 0, 0);
        }
      }
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < MB; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            tot[i][j][e] = __builtin_fmaf(16.0f * sc[i][s], __builtin_fmaf(-zp[i][s], sum[j][e], acc[i][j][e]), tot[i][j][e]);
    }
  }
  // lane (r, g) holds column r, rows 4 g .. 4 g + 3
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < MB; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) red[w][(16 * j + 4 * g + e) * LD + 16 * i + r] = tot[i][j][e];
  __syncthreads();
  for (int t = threadIdx.x; t < 16 * NB * 16 * MB; t += 64 * KW) {
    const int m = t / (16 * NB), n = t % (16 * NB);
    if (m0 + m >= p.M || n0 + n >= p.N) continue;
    float v = red[0][m * LD + n];
#pragma unroll
    for (int i = 1; i < KW; ++i) v += red[i][m * LD + n];
    if (p.bias != nullptr) v += p.bias[n0 + n];
    p.y[static_cast<int64_t>(m0 + m) * p.ldy + n0 + n] = static_cast<bf16>(apply_act_rt(v, p.act));
  }
}

// int8 codes in -8..7 [N, K] -> packed rows; one word per thread.  Codes past
// K are zero (nibble 8).
__global__ __launch_bounds__(256) void w4_pack(const int8_t *q, uint32_t *out, int64_t words, int K) {
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (at >= words) return;
  const int per_row = (K + 127) / 128 * 16;
  const int64_t n = at / per_row;
  const int word = static_cast<int>(at - n * per_row), i = word & 15;
  const int k0 = (word >> 4) * 128 + 32 * (i & 3) + 8 * (i >> 2);
  uint32_t v = 0;
  for (int j = 0; j < 8; ++j) {
    const int code = k0 + j < K ? q[n * K + k0 + j] : 0;
    v |= static_cast<uint32_t>((code + 8) & 15) << (4 * w4_nibble(j));
  }
  out[at] = v;
}

// Packed weights -> bf16 [N, K], rounded once; one word per thread.
template <bool ZERO>
__global__ __launch_bounds__(256) void w4_unpack(W4Args p, bf16 *out, int64_t words) {
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (at >= words) return;
  const int per_row = (p.K + 7) / 8, chunks = (p.K + 127) / 128;
  const int64_t n = at / per_row;
  const int word = static_cast<int>(at - n * per_row), k0 = 8 * word;
  const int c = (word >> 2) & 3, g = word & 3;
  const uint32_t v = reinterpret_cast<const uint32_t *>(p.w)[(n * chunks + (word >> 4)) * 16 + 4 * g + c];
  const int64_t grp = n * p.groups + k0 / p.group;
  const float sc = p.scale[grp];
  const int off = 8 + (ZERO ? p.zero[grp] : 0);
  bf16x8 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bf16x2 pr = cvt_pk_bf16(static_cast<float>(static_cast<int>((v >> (4 * w4_nibble(2 * j))) & 15u) - off) * sc,
                                  static_cast<float>(static_cast<int>((v >> (4 * w4_nibble(2 * j + 1))) & 15u) - off) * sc);
    r[2 * j] = pr[0];
    r[2 * j + 1] = pr[1];
  }
  *reinterpret_cast<bf16x8 *>(out + n * p.K + k0) = r;
}

template <int MB, int NB, int SUB, int KW>
inline void launch_gemm_w4(const W4Args &p, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(cdiv(p.N, 16 * NB)), static_cast<unsigned>(cdiv(p.M, 16 * MB)));
  if (p.zero) hipLaunchKernelGGL((gemm_w4<MB, NB, SUB, KW, true>), grid, dim3(64 * KW), 0, s, p);
  else hipLaunchKernelGGL((gemm_w4<MB, NB, SUB, KW, false>), grid, dim3(64 * KW), 0, s, p);
}

template <int MB, int NB, int KW>
inline void launch_gemm_w4(const W4Args &p, hipStream_t s) {
  if (p.group == 32) launch_gemm_w4<MB, NB, 4, KW>(p, s);
  else if (p.group == 64) launch_gemm_w4<MB, NB, 2, KW>(p, s);
  else launch_gemm_w4<MB, NB, 1, KW>(p, s);
}

inline void launch_gemm_w4(const W4Args &p, hipStream_t s) {
  if (p.M <= 16) launch_gemm_w4<1, 1, 8>(p, s);
  else if (p.M <= 32) launch_gemm_w4<2, 1, 8>(p, s);
  else launch_gemm_w4<4, 1, 8>(p, s);
}

}  // namespace teeny
