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
// (An infinity in a row of x makes both sums infinite, and the row's outputs NaN.)
#pragma once

#include "mfma.hpp"

#include <algorithm>
#include <type_traits>

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
  int chunks_per_group;  // group / 128, and 2^32 over it rounded up
  uint32_t magic;
  int vec;               // a chunk's scales and zero points are aligned vectors
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
// columns and up to XR rows of x (blockIdx.y); its KW waves share out the
// chunks of K and meet in LDS in wave order.  The weights come straight from
// memory in their operand's layout, a round of U chunks ahead.  What else a
// chunk needs is small but touches more cache lines than they do: a lane's
// scales for one chunk are a few bytes of 16 rows, so lane group g loads those
// of chunk c + g, four chunks in one go, and hands them round in LDS; x is read
// in whole rows of 256 bytes and turned there too.  (us, 11008 x 4096 with one
// row, and 4096 x 4096 with 16 and groups of 32 with zero points: scales and x
// straight into the lanes that use them 10.6 and 14.1, of which the scales were
// 2.1 and 7.5; so 8.3 and 7.6.  Reading the weights alone takes 4.5 and 2.5.)
// The loop stays rolled: unrolled over four chunks the code, which each wave
// runs but once, took longer to fetch (11.7 and 10.1).  Past a wave's share a
// round takes the share's last chunk again, with scale 0.  SUB: groups per chunk.
template <int XR, int NB, int SUB, int KW, int U, bool ZERO>
__global__ __launch_bounds__(64 * KW) void gemm_w4(W4Args p) {
  static_assert(SUB == 1 || SUB == 2 || SUB == 4, "groups of a 128-k chunk");
  static_assert(4 % U == 0, "a round's chunks lie in one set of four");
  constexpr int MB = (XR + 15) / 16, NX = XR / 4;  // blocks of 16 rows, 16-byte vectors of x per lane and chunk
  constexpr int LX = 128 + 8;                      // row stride of the x tile: no bank conflicts over 16 rows
  constexpr int LD = 16 * NB + 1;
  constexpr int XT = 16 * MB * LX / 2, RED = 16 * MB * LD, ST = (ZERO ? 2 : 1) * NB * 64 * SUB;  // 4-byte words
  __shared__ __attribute__((aligned(16))) float lds[KW * (XT + ST > RED ? XT + ST : RED)];
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16 * NB, m0 = blockIdx.y * 16 * MB;
  const int chunks = (p.K + 127) / 128, per = (chunks + KW - 1) / KW;
  const int cb = __builtin_amdgcn_readfirstlane(min(chunks, w * per));
  const int ce = __builtin_amdgcn_readfirstlane(min(chunks, cb + per));
  bf16 *xt = reinterpret_cast<bf16 *>(lds + w * (XT + ST));
  float *st = lds + w * (XT + ST) + XT;
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
  const bf16 *xrow[NX];
#pragma unroll
  for (int i = 0; i < NX; ++i) xrow[i] = p.x + static_cast<int64_t>(min(m0 + 4 * i + g, p.M - 1)) * p.K;

  f32x4 tot[NB][MB];
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < MB; ++j) tot[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  // chunks c .. c + U - 1: weights, and x in whole rows.  Past the wave's share: the share's last chunk, with scale 0.
  struct Round {
    u32x4 q[U][NB], x[U][NX];
  };
  struct Scales {  // of chunk c + g, SUB groups
    float sc[NB][SUB];
    int32_t zp[NB][ZERO ? SUB : 1];
  };
  auto load = [&](Round &a, int c0) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = min(c0 + u, ce - 1);
#pragma unroll
      for (int i = 0; i < NB; ++i) a.q[u][i] = *reinterpret_cast<const u32x4 *>(wrow[i] + 64 * static_cast<int64_t>(c));
      // zeros past K, a multiple of 8: a vector is inside or outside as a whole
      const int k = 128 * c + 8 * r;
      const bool in = k < p.K;
#pragma unroll
      for (int i = 0; i < NX; ++i) {
        a.x[u][i] = *reinterpret_cast<const u32x4 *>(xrow[i] + (in ? k : 0));
        if (!in) a.x[u][i] = u32x4{0u, 0u, 0u, 0u};
      }
    }
  };
  auto load_scales = [&](Scales &a, int c0) __attribute__((always_inline)) {
    const int c = min(c0 + g, ce - 1);
    const int at = SUB > 1 ? c * SUB : p.chunks_per_group == 1 ? c : static_cast<int>(__umulhi(c, p.magic));
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      if (SUB > 1 && p.vec) {  // a chunk's scales are one aligned vector
        __builtin_memcpy(a.sc[i], __builtin_assume_aligned(srow[i] + at, 4 * SUB), 4 * SUB);
        if constexpr (ZERO) __builtin_memcpy(a.zp[i], __builtin_assume_aligned(zrow[i] + at, 4 * SUB), 4 * SUB);
      } else {
#pragma unroll
        for (int s = 0; s < SUB; ++s) {  // groups past the last one hold no k
          a.sc[i][s] = srow[i][min(at + s, p.groups - 1)];
          if constexpr (ZERO) a.zp[i][s] = zrow[i][min(at + s, p.groups - 1)];
        }
      }
      if (c0 + g >= ce)
#pragma unroll
        for (int s = 0; s < SUB; ++s) a.sc[i][s] = 0.0f;
    }
  };
  const uint32_t one = 0x3F803F80u;
  const bf16x8 ones = __builtin_bit_cast(bf16x8, (u32x4{one, one, one, one}));
  if (cb < ce) {
    Round next;
    Scales snext;
    load_scales(snext, cb);
    load(next, cb);
#pragma unroll 1
    for (int c = cb; c < ce; c += U) {
      const Round now = next;
      __builtin_amdgcn_wave_barrier();
      if (((c - cb) & 3) == 0) {  // four chunks' scales at a time, [chunk][row][group]
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
          for (int s = 0; s < SUB; ++s) {
            st[(i * 64 + lane) * SUB + s] = snext.sc[i][s];
            if constexpr (ZERO) st[(NB + i) * 64 * SUB + lane * SUB + s] = 1.5f + static_cast<float>(snext.zp[i][s]) * 0.0625f;
          }
        if (c + 4 < ce) load_scales(snext, c + 4);
      }
      if (c + U < ce) load(next, c + U);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < NX; ++i) *reinterpret_cast<u32x4 *>(xt + (4 * i + g) * LX + 8 * r) = now.x[u][i];
        // the wave's lanes read what its other lanes wrote
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        const float *sat = st + (((c + u - cb) & 3) * 16 + r) * SUB;
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
            bf16x8 x[MB];
#pragma unroll
            for (int j = 0; j < MB; ++j) {
              // (rows past XR hold nothing and are not stored)
              x[j] = *reinterpret_cast<const bf16x8 *>(xt + (16 * j + (XR < 16 ? r % XR : r)) * LX + 32 * t + 8 * g);
              sum[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[j], ones, sum[j], 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < NB; ++i) {
              const bf16x8 b = w4_values(now.q[u][i][t]);
#pragma unroll
              for (int j = 0; j < MB; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[j], b, acc[i][j], 0, 0, 0);
            }
          }
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            const float sc = sat[i * 64 * SUB + s], zp = ZERO ? sat[(NB + i) * 64 * SUB + s] : 1.5f;
#pragma unroll
            for (int j = 0; j < MB; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                tot[i][j][e] = __builtin_fmaf(sc, __builtin_fmaf(-zp, sum[j][e], acc[i][j][e]), tot[i][j][e]);
          }
        }
      }
    }
  }
  __syncthreads();
  // lane (r, g) holds column r, rows 4 g .. 4 g + 3
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < MB; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) lds[w * RED + (16 * j + 4 * g + e) * LD + 16 * i + r] = tot[i][j][e];
  __syncthreads();
  for (int t = threadIdx.x; t < 16 * NB * XR; t += 64 * KW) {
    const int m = t / (16 * NB), n = t % (16 * NB);
    if (m0 + m >= p.M || n0 + n >= p.N) continue;
    float v = lds[m * LD + n];
#pragma unroll
    for (int i = 1; i < KW; ++i) v += lds[i * RED + m * LD + n];
    v *= 16.0f;
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

// Packed weights -> bf16 [N, K], rounded once (group scales do not come out of the
// tiles' sums over all of K): the rms error against 64 bits goes from 0.0017, the
// output's own rounding, to 0.0023.  One word per thread.  11008 x 4096 take 21 us,
// 113 MB: the copy rate.
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

template <int XR, int NB, int SUB, int KW, int U>
inline void launch_w4_groups(W4Args p, hipStream_t s) {
  p.chunks_per_group = std::max(1, p.group / 128);
  p.magic = static_cast<uint32_t>((int64_t{1} << 32) / p.chunks_per_group + 1);  // exact below 2^16 chunks
  p.vec = p.groups % SUB == 0 && aligned(p.scale, 4 * SUB) && aligned(p.zero, 4 * SUB);
  const dim3 grid(static_cast<unsigned>(cdiv(p.N, 16 * NB)), static_cast<unsigned>(cdiv(p.M, (XR + 15) / 16 * 16)));
  if (p.zero) hipLaunchKernelGGL((gemm_w4<XR, NB, SUB, KW, U, true>), grid, dim3(64 * KW), 0, s, p);
  else hipLaunchKernelGGL((gemm_w4<XR, NB, SUB, KW, U, false>), grid, dim3(64 * KW), 0, s, p);
}

template <int XR, int NB, int KW, int U>
inline void launch_w4_form(const W4Args &p, hipStream_t s) {
  if (p.group == 32) launch_w4_groups<XR, NB, 4, KW, U>(p, s);
  else if (p.group == 64) launch_w4_groups<XR, NB, 2, KW, U>(p, s);
  else launch_w4_groups<XR, NB, 1, KW, U>(p, s);
}

// Rows of x and blocks of columns per workgroup, and waves along K.  In us, the
// weights through 4 to 6 sets of operands.  Sixteen waves pay once each has several
// rounds: 8 x 4096 x 11008 11.0 / 9.2, 16 x 2048 x 8192 9.5 / 8.5, but 8 x 4096 x
// 4096 7.0 / 8.3.  Nine rows and more with over three workgroups of 16 columns to
// a CU take 32 columns each: 16 x 16000 x 4096 13.4 / 11.9, but 16 x 11008 x 4096 10.6
// / 10.9 and 8 x 16000 x 4096 11.4 / 11.6.  Past 16 rows two column blocks share what is read of x, and the
// number of workgroups decides.  Registers let two of eight waves onto a CU, one
// with 32 rows, and a second turn costs the most: 16 rows while that is one a CU,
// else 32 while that is; beyond, workgroups of four waves, of which four or two
// (32 rows) fit.  16 rows / 32 / 16 of four waves / 32 of four: 32 x 4096 x 4096
// 7.1 / 9.1 / 9.4 / 11.6, 32 x 5504 x 2048 8.1 / 6.9 / 8.3 / 7.7, 64 x 4096 x 4096
// 10.8 / 9.5 / 12.1 / 11.8, 50 x 5504 x 2048 10.8 / 12.5 / 10.0 / 10.3, 32 x 11008 x
// 4096 15.2 / 17.1 / 15.6 / 16.3, 64 x 7000 x 4096 19.9 / 18.1 / 20.1 / 17.1, 64 x
// 11008 x 4096 26.3 / 25.0 / 27.1 / 21.2, 150 x 11008 x 4096 56 / 56 / 56 / 44.
inline void launch_gemm_w4(const W4Args &p, hipStream_t s) {
  const bool deep = p.K >= 8192;
  const int64_t cols = cdiv(p.N, 32), cus = device_cu_count();
  if (p.M <= 16) {
    if (p.M <= 4) deep ? launch_w4_form<4, 1, 16, 2>(p, s) : launch_w4_form<4, 1, 8, 2>(p, s);
    else if (p.M <= 8) deep ? launch_w4_form<8, 1, 16, 1>(p, s) : launch_w4_form<8, 1, 8, 1>(p, s);
    else if (deep) launch_w4_form<16, 1, 16, 1>(p, s);
    else cols * 2 > 3 * cus ? launch_w4_form<16, 2, 8, 1>(p, s) : launch_w4_form<16, 1, 8, 1>(p, s);
  } else {
    const int64_t wgs = cols * cdiv(p.M, 32);
    if (cols * cdiv(p.M, 16) <= cus) launch_w4_form<16, 2, 8, 1>(p, s);
    else if (wgs <= cus) launch_w4_form<32, 2, 8, 1>(p, s);
    else if (2 * wgs <= 3 * cus) launch_w4_form<16, 2, 4, 1>(p, s);
    else launch_w4_form<32, 2, 4, 1>(p, s);
  }
}

}  // namespace teeny
