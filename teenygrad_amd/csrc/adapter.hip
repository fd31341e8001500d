// Low-rank adapters of many requests beside a projection that they share:
//
//   out[m] = y[m] + B[a] (scale[a] A[a] x[m]),  a = adapters[m] (none: out[m] = y[m])
//
// x bf16 [M, K], A bf16 [adapters, rank, K], B bf16 [adapters, N, rank], y and out
// bf16 [M, N].  The reference has no such operator; the shared projection is
// teeny_linear_forward's (kernels/teeny-kernels/src/nn/mlp/linear.rs:20-116) or one
// of its quantized forms.
#include "mfma.hpp"

#include <algorithm>

namespace teeny {

struct AdapterArgs {
  const bf16 *x, *a, *b;
  const int32_t *ids;
  const float *scale;
  const bf16 *y;
  bf16 *out;
  int64_t x_stride, y_stride, out_stride;
  int M, N, K, rank, adapters;
  int cols;                          // output columns of a workgroup
  float *part;                       // [splits][M][RP] products of the ranks, RP: the rank in whole tiles of 16
  int splits, chunk, slots;          // chunk: k's of a split; slots: workgroups to a tile of rows, 0: one to each row
};

__device__ __forceinline__ f32x4 mfma_16x16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
// Eight numbers of a row.  Rows may begin anywhere (global memory takes 16 bytes at any address).
__device__ __forceinline__ u32x4 adapter_load(const AdapterArgs &p, int m, int n) {
  u32x4 v;
  __builtin_memcpy(&v, p.y + m * p.y_stride + n, 16);
  return v;
}
__device__ __forceinline__ void adapter_store(const AdapterArgs &p, int m, int n, u32x4 v, f32x4 lo, f32x4 hi) {
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x4 &a = i < 2 ? lo : hi;
    o[i] = __builtin_bit_cast(uint32_t, cvt_pk_bf16(__uint_as_float(v[i] << 16) + a[2 * (i & 1)],
                                                    __uint_as_float(v[i] & 0xffff0000u) + a[2 * (i & 1) + 1]));
  }
  typedef u32x4 any __attribute__((aligned(2)));
  // past the caches, which hold B (2000 rows x 11008 columns of rank 64: 36.0 -> 30.0 us)
  __builtin_nontemporal_store(o, reinterpret_cast<any *>(p.out + m * p.out_stride + n));
}
// Where the 64 columns pass the last one: number by number; rows as offsets from m0's, so that the 16 addresses are one.
__device__ __forceinline__ void adapter_edge(const AdapterArgs &p, int m0, int row, int n, const f32x4 (&add)[4]) {
  const int extent = min(p.M - m0, 32) - 1;  // of a workgroup's rows, two tiles at most
  const auto yr = buffer_rsrc(p.y + m0 * p.y_stride, static_cast<int>((extent * p.y_stride + p.N) * 2));
  const auto outr = buffer_rsrc(p.out + m0 * p.out_stride, static_cast<int>((extent * p.out_stride + p.N) * 2));
  const int y_at = static_cast<int>((row * p.y_stride + n) * 2), out_at = static_cast<int>((row * p.out_stride + n) * 2);
  uint16_t v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __builtin_amdgcn_raw_buffer_load_b16(yr, y_at + 64 * (i >> 3) + 2 * (i & 7), 0, 0);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int at = 32 * (i >> 3) + (i & 7);
    const bf16 o = static_cast<bf16>(__uint_as_float(static_cast<uint32_t>(v[i]) << 16) + add[i >> 2][i & 3]);
    __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, o), outr, n + at < p.N ? out_at + 2 * at : kOffNone, 0, 0);
  }
}
// Columns n0 .. n1 - 1 of rows without an adapter, by the workgroup.
__device__ __forceinline__ void adapter_copy(const AdapterArgs &p, int m0, uint64_t rows, int n0, int n1) {
#pragma unroll 1
  for (; rows != 0; rows &= rows - 1) {
    const int m = m0 + __builtin_ctzll(rows);
    const bf16 *y = p.y + m * p.y_stride;
    bf16 *out = p.out + m * p.out_stride;
#pragma unroll 1
    for (int n = n0 + 8 * threadIdx.x; n < n1; n += 8 * blockDim.x) {
      if (n + 8 <= n1) {
        __builtin_memcpy(out + n, y + n, 16);
      } else {
#pragma unroll 1
        for (int i = n; i < n1; ++i) out[i] = y[i];
      }
    }
  }
}
// Whether one of a lane's sums is NaN.  An infinity in B gives NaN beside a second part that is 0 or of the other sign,
// where the first part alone gives what the whole number does: those sums are made again without the second part.
__device__ __forceinline__ bool adapter_nan(f32x4 o) { return __builtin_isunordered(o[0], o[1]) | __builtin_isunordered(o[2], o[3]); }
__device__ __forceinline__ void adapter_mend(f32x4 &o, f32x4 first) {
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = o[i] == o[i] ? o[i] : first[i];
}
// The row of B that lane c holds for tile j of the columns n ..: a lane's products are a row's columns n + 8 g + 0..7, and 32 further on.
__device__ __forceinline__ int adapter_col(int n, int j, int c) { return n + 32 * (j >> 1) + 8 * (c >> 2) + 4 * (j & 1) + (c & 3); }

// Lanes of two rows swap halves: each then has the same eight columns of both (odd lanes those 32 further on), and a wave's
// access is 128 bytes of each row, a whole line where rows begin on one.
__device__ __forceinline__ float dpp_swap(float v) {  // lane l has lane l ^ 1's
  return __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(v), 0xb1, 0xf, 0xf, false));
}
__device__ __forceinline__ void adapter_swap(f32x4 (&o)[4], bool odd) {
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float low = o[j][i], high = o[2 + j][i];
      const float other_low = dpp_swap(low), other_high = dpp_swap(high);
      o[j][i] = odd ? other_high : low;
      o[2 + j][i] = odd ? high : other_low;
    }
}

// The rows of 16 MT ones that each adapter has: lane l's row l.  Either (slots 0) there is a workgroup for each row, which
// takes the adapter of which the row is the first, or `slots` workgroups for each tile take its adapters in turn.
template <int MT>
struct AdapterRows {
  int m0, id;     // the first row; the lane's adapter (-1: none, -2: no row)
  uint64_t left;  // rows whose adapters no workgroup has taken yet
  int skip;       // adapters of other workgroups before the next one
  __device__ __forceinline__ AdapterRows(const AdapterArgs &p, int block) {
    // the first workgroups of all tiles, then the second ones, of which few may have anything to do: each XCD has its share
    const int lane = threadIdx.x & 63, tiles = (p.M + 16 * MT - 1) / (16 * MT);
    skip = p.slots == 0 ? 0 : block / tiles;
    m0 = (p.slots == 0 ? block / (16 * MT) : block - skip * tiles) * 16 * MT;
    id = -2;
    if (lane < 16 * MT && m0 + lane < p.M) {
      id = p.ids[m0 + lane];
      if (id < 0 || id >= p.adapters) id = -1;
    }
    left = __ballot(id >= -1);
    if (p.slots == 0) {
      const uint64_t same = __ballot(id == __builtin_amdgcn_readlane(id, block - m0));
      left = __builtin_ctzll(same) == block - m0 ? same : 0;
    }
  }
  // whether there is another adapter for this workgroup; it and its rows
  __device__ __forceinline__ bool next(const AdapterArgs &p, int &a, uint64_t &rows) {
    while (left != 0) {
      a = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
      rows = __ballot(id == a);
      left &= ~rows;
      if (skip-- == 0) {
        skip = p.slots - 1;
        return true;
      }
    }
    return false;
  }
};

// part[split] = A[a] x over the split's k's.  Four waves share them out in turn, 64 at
// a time, and meet in LDS; all of a wave's share is in flight at once (a k past the
// split's end loads zeros).  Rows of other adapters are multiplied too and not
// written; rows of A past the rank repeat the last one and are not read again.  Bound
// by latency: ids, operands, the meeting, in turn.  64 requests, 40 adapters of rank
// 16, K 4096: 5 us; 2000 rows of rank 64: 12 us, 35 MB read.
template <int RT, int MT>
__global__ __launch_bounds__(256) void adapter_down(AdapterArgs p) {
  constexpr int U = RT * MT >= 8 ? 2 : 4, RP = 16 * RT;
  __shared__ __attribute__((aligned(16))) float sum[4][16 * MT][RP + 4];
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, c = lane & 15, g = lane >> 4;
  AdapterRows<MT> rows(p, blockIdx.x);
  const int kb = blockIdx.y * p.chunk, ke = min(p.K, kb + p.chunk);
  const int last = min(16 * MT, p.M - rows.m0) - 1;
  const auto xr = buffer_rsrc(p.x + rows.m0 * p.x_stride, static_cast<int>((last * p.x_stride + p.K) * 2));
  int x_at[MT], a_at[RT];
#pragma unroll
  for (int t = 0; t < MT; ++t) x_at[t] = static_cast<int>((min(16 * t + c, last) * p.x_stride + 8 * g) * 2);
#pragma unroll
  for (int t = 0; t < RT; ++t) a_at[t] = (min(16 * t + c, p.rank - 1) * p.K + 8 * g) * 2;
  int a;
  uint64_t mine;
  while (rows.next(p, a, mine)) {
    if (a < 0) continue;
    const auto ar = buffer_rsrc(p.a + static_cast<int64_t>(a) * p.rank * p.K, p.rank * p.K * 2);
    f32x4 acc[RT][MT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[r][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int k = kb + 64 * w; k < ke; k += 256 * U) {
      u32x4 xf[U][2][MT], af[U][2][RT];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int at = k + 256 * u + 32 * h;
          const bool in = at + 8 * g < ke;
#pragma unroll
          for (int r = 0; r < RT; ++r) af[u][h][r] = buffer_load16(ar, in ? a_at[r] + 2 * at : kOffNone);
#pragma unroll
          for (int t = 0; t < MT; ++t) xf[u][h][t] = buffer_load16(xr, in ? x_at[t] + 2 * at : kOffNone);
        }
      __builtin_amdgcn_sched_barrier(0);  // or products are moved up between the loads, to save registers
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int t = 0; t < MT; ++t)
              acc[r][t] = mfma_16x16(__builtin_bit_cast(bf16x8, af[u][h][r]), __builtin_bit_cast(bf16x8, xf[u][h][t]), acc[r][t]);
    }
    __syncthreads();  // the last adapter's sums have been read
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int r = 0; r < RT; ++r) *reinterpret_cast<f32x4 *>(&sum[w][16 * t + c][16 * r + 4 * g]) = acc[r][t];
    __syncthreads();
    for (int i = tid; i < 16 * MT * RP / 4; i += 256) {
      const int m = i / (RP / 4), r = 4 * (i - m * (RP / 4));
      if (!((mine >> m) & 1)) continue;
      f32x4 v = *reinterpret_cast<const f32x4 *>(&sum[0][m][r]);
#pragma unroll
      for (int j = 1; j < 4; ++j) v += *reinterpret_cast<const f32x4 *>(&sum[j][m][r]);
      *reinterpret_cast<f32x4 *>(p.part + (static_cast<int64_t>(blockIdx.y) * p.M + rows.m0 + m) * RP + r) = v;
    }
  }
}

// out = y + B[a] (scale part).  A wave takes 64 columns a time.  The ranks' products
// are two bf16 parts of an fp32 number; at a rank of 16 or less both are the k's of
// one product.  The next columns' operands are loaded as soon as this one's have
// been multiplied, the first ones ahead of the ranks' sums.  Those 64 requests with
// 11008 columns: 6 us, ids, parts and B in turn; 2000 rows of rank 64: 28 us, 88 MB of
// y and out at 3.1 TB/s.  (With an XCD's workgroups on one range of columns, so that
// each reads its part of B alone: 46 us for both launches to 40.6.)
template <int RT, int MT>
__global__ __launch_bounds__(256, RT * MT >= 16 ? 1 : RT * MT >= 8 ? 2 : RT * MT >= 4 || MT == 2 ? 3 : 4) void adapter_up(AdapterArgs p) {
  constexpr int RP = 16 * RT, KS = RT == 1 ? 1 : RT / 2, LH = (RT == 1 ? 32 : RP) + 8, PARTS = RT == 1 ? 1 : 2;
  __shared__ __attribute__((aligned(16))) bf16 hs[PARTS][16 * MT][LH];
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, c = lane & 15, g = lane >> 4;
  AdapterRows<MT> rows(p, blockIdx.x);
  const int n0 = blockIdx.y * p.cols, n1 = min(p.N, n0 + p.cols);
  int a;
  uint64_t mine;
  while (rows.next(p, a, mine)) {
    if (a < 0) {
      if (p.out != p.y) adapter_copy(p, rows.m0, mine, n0, n1);
      continue;
    }
    int cc = c, gg = g;
    asm volatile("" : "+v"(cc), "+v"(gg));
    const auto br = buffer_rsrc(p.b + static_cast<int64_t>(a) * p.N * p.rank, p.N * p.rank * 2);
    const int r0 = RT == 1 ? 8 * (gg & 1) : 8 * gg;
    u32x4 b[4][KS];
    u32x4 y[MT][2];
    const bool odd = cc & 1;
    const int pair = cc & ~1, nn = 8 * gg + 32 * (cc & 1);  // the rows and columns that a lane has in the end
    bool in[MT][2];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int q = 0; q < 2; ++q) in[t][q] = (mine >> (16 * t + pair + q)) & 1;
    uint32_t b_at[KS];  // zeros past the rank
#pragma unroll
    for (int k = 0; k < KS; ++k) b_at[k] = r0 + 32 * k < p.rank ? 2 * (r0 + 32 * k) : static_cast<uint32_t>(kOffNone);
    auto load_b = [&](int n) __attribute__((always_inline)) {  // and past the columns
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int k = 0; k < KS; ++k)
          b[j][k] = buffer_load16(br, static_cast<int>(b_at[k] + 2 * static_cast<uint32_t>(adapter_col(n, j, cc) * p.rank)));
    };
    auto load_y = [&](int n) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int q = 0; q < 2; ++q)
          if (in[t][q]) y[t][q] = adapter_load(p, rows.m0 + 16 * t + pair + q, n + nn);
    };
    auto products = [&](int t, f32x4 (&o)[4]) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        o[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < PARTS; ++s)
#pragma unroll
          for (int k = 0; k < KS; ++k)
            o[j] = mfma_16x16(__builtin_bit_cast(bf16x8, b[j][k]),
                              *reinterpret_cast<const bf16x8 *>(&hs[s][16 * t + cc][32 * k + 8 * gg]), o[j]);
      }
      if (__builtin_expect(__any(adapter_nan(o[0]) | adapter_nan(o[1]) | adapter_nan(o[2]) | adapter_nan(o[3])), 0)) {
        const u32x4 zero = {};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f32x4 first = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int k = 0; k < KS; ++k)
            first = mfma_16x16(__builtin_bit_cast(bf16x8, RT > 1 || gg < 2 ? b[j][k] : zero),
                               *reinterpret_cast<const bf16x8 *>(&hs[0][16 * t + cc][32 * k + 8 * gg]), first);
          adapter_mend(o[j], first);
        }
      }
    };
    int n = n0 + 64 * w;
    asm volatile("" : "+s"(n));  // or the loop over adapters carries every address along
    const int n_whole = n1 - 63;  // below it all of 64 columns are there (a range that is not the last has whole ones)
    if (n < n1) load_b(n);
    if (n < n_whole) load_y(n);
    const float scale = p.scale != nullptr ? p.scale[a] : 1.0f;
    __syncthreads();  // the last adapter's products have been read
    for (int i = tid; i < 4 * MT * RP; i += 256) {
      const int row = i / (RP / 4), r = 4 * (i - row * (RP / 4));
      f32x4 h = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (r < p.rank && ((mine >> row) & 1)) {  // the rank is a multiple of 8
        const float *at = p.part + static_cast<int64_t>(rows.m0 + row) * RP + r;
        const int64_t next = static_cast<int64_t>(p.M) * RP;
#pragma unroll 4
        for (int s = 0; s < p.splits; ++s) h += *reinterpret_cast<const f32x4 *>(at + s * next);
        h *= scale;
      }
      bf16x4 hi, lo;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        hi[e] = static_cast<bf16>(h[e]);
        lo[e] = fabsf(static_cast<float>(hi[e])) < INFINITY ? static_cast<bf16>(h[e] - static_cast<float>(hi[e])) : static_cast<bf16>(0.0f);
      }
      *reinterpret_cast<bf16x4 *>(&hs[0][row][r]) = hi;
      *reinterpret_cast<bf16x4 *>(RT == 1 ? &hs[0][row][16 + r] : &hs[PARTS - 1][row][r]) = lo;
    }
    __syncthreads();
    for (; n < n_whole; n += 256) {
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        f32x4 o[4];
        products(t, o);
        if (t == MT - 1 && n + 256 < n1) load_b(n + 256);
        adapter_swap(o, odd);
#pragma unroll
        for (int q = 0; q < 2; ++q)
          if (in[t][q]) {
            adapter_store(p, rows.m0 + 16 * t + pair + q, n + nn, y[t][q], o[2 * q], o[2 * q + 1]);
            if (n + 256 < n_whole) y[t][q] = adapter_load(p, rows.m0 + 16 * t + pair + q, n + 256 + nn);
          }
      }
    }
    if (n < n1) {
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        f32x4 o[4];
        products(t, o);
        if ((mine >> (16 * t + cc)) & 1) adapter_edge(p, rows.m0, 16 * t + cc, n + 8 * gg, o);
      }
    }
  }
}

// Both products in one launch, without scratch: each workgroup has the ranks' products
// of its rows to itself, so A is read once for each range of columns.  Sixteen waves
// share out the k's, then the columns, 16 at a time.
template <int RT>
__global__ __launch_bounds__(1024) void adapter_one(AdapterArgs p) {
  constexpr int U = RT == 1 ? 4 : RT == 2 ? 2 : 1, H = RT == 8 ? 1 : 2, RP = 16 * RT, KS = RT == 1 ? 1 : RT / 2, LH = (RT == 1 ? 32 : RP) + 8, PARTS = RT == 1 ? 1 : 2;
  __shared__ __attribute__((aligned(16))) float sum[16][16][RP + 4];
  __shared__ __attribute__((aligned(16))) bf16 hs[PARTS][16][LH];
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, c = lane & 15, g = lane >> 4;
  AdapterRows<1> rows(p, blockIdx.x);
  const int n0 = blockIdx.y * p.cols, n1 = min(p.N, n0 + p.cols);
  const int last = min(16, p.M - rows.m0) - 1;
  const auto xr = buffer_rsrc(p.x + rows.m0 * p.x_stride, static_cast<int>((last * p.x_stride + p.K) * 2));
  const int x_at = static_cast<int>((min(c, last) * p.x_stride + 8 * g) * 2);
  int a;
  uint64_t mine;
  while (rows.next(p, a, mine)) {
    if (a < 0) {
      if (p.out != p.y) adapter_copy(p, rows.m0, mine, n0, n1);
      continue;
    }
    const bool in = (mine >> c) & 1;
    const auto ar = buffer_rsrc(p.a + static_cast<int64_t>(a) * p.rank * p.K, p.rank * p.K * 2);
    const auto br = buffer_rsrc(p.b + static_cast<int64_t>(a) * p.N * p.rank, p.N * p.rank * 2);
    f32x4 acc[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) acc[r] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int k = 64 * w; k < p.K; k += 1024 * U) {
#pragma unroll 1
      for (int h0 = 0; h0 < 2; h0 += H) {
        u32x4 xf[U][H], af[U][H][RT];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int h = 0; h < H; ++h) {
            const int at = k + 1024 * u + 32 * (h0 + h);
            const bool there = at + 8 * g < p.K;
#pragma unroll
            for (int r = 0; r < RT; ++r)
              af[u][h][r] = buffer_load16(ar, there ? (min(16 * r + c, p.rank - 1) * p.K + at + 8 * g) * 2 : kOffNone);
            xf[u][h] = buffer_load16(xr, there ? x_at + 2 * at : kOffNone);
          }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int h = 0; h < H; ++h)
#pragma unroll
            for (int r = 0; r < RT; ++r)
              acc[r] = mfma_16x16(__builtin_bit_cast(bf16x8, af[u][h][r]), __builtin_bit_cast(bf16x8, xf[u][h]), acc[r]);
      }
    }
    // the first columns' operands, ahead of the sums
    const int r0 = RT == 1 ? 8 * (g & 1) : 8 * g;
    u32x4 b[KS];
    auto load_b = [&](int n) __attribute__((always_inline)) {  // zeros past the rank and the columns
#pragma unroll
      for (int k = 0; k < KS; ++k) 
        b[k] = buffer_load16(br, static_cast<int>(r0 + 32 * k < p.rank ? (static_cast<uint32_t>((n + c) * p.rank) + r0 + 32 * k) * 2u : kOffNone));
    };
    int n = n0 + 16 * w;
    if (n < n1) load_b(n);
    const float scale = p.scale != nullptr ? p.scale[a] : 1.0f;
    __syncthreads();  // the last adapter's products have been read
#pragma unroll
    for (int r = 0; r < RT; ++r) *reinterpret_cast<f32x4 *>(&sum[w][c][16 * r + 4 * g]) = acc[r];
    __syncthreads();
    for (int i = tid; i < 16 * RP; i += 1024) {
      const int m = i / RP, r = i - m * RP;
      float h = 0.0f;
      if ((mine >> m) & 1 && r < p.rank) {
#pragma unroll
        for (int j = 0; j < 16; ++j) h += sum[j][m][r];
        h *= scale;
      }
      const bf16 hi = static_cast<bf16>(h);
      hs[0][m][r] = hi;
      hs[PARTS - 1][m][RT == 1 ? 16 + r : r] = fabsf(static_cast<float>(hi)) < INFINITY ? static_cast<bf16>(h - static_cast<float>(hi)) : static_cast<bf16>(0.0f);
    }
    __syncthreads();
    for (; n < n1; n += 256) {
      f32x4 o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < PARTS; ++s)
#pragma unroll
        for (int k = 0; k < KS; ++k)
          o = mfma_16x16(__builtin_bit_cast(bf16x8, b[k]), *reinterpret_cast<const bf16x8 *>(&hs[s][c][32 * k + 8 * g]), o);
      if (__builtin_expect(__any(adapter_nan(o)), 0)) {
        const u32x4 zero = {};
        f32x4 first = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < KS; ++k)
          first = mfma_16x16(__builtin_bit_cast(bf16x8, RT > 1 || g < 2 ? b[k] : zero),
                             *reinterpret_cast<const bf16x8 *>(&hs[0][c][32 * k + 8 * g]), first);
        adapter_mend(o, first);
      }
      if (n + 256 < n1) load_b(n + 256);
      if (in) {
        const bf16 *y = p.y + (rows.m0 + c) * p.y_stride + n + 4 * g;
        bf16 *out = p.out + (rows.m0 + c) * p.out_stride + n + 4 * g;
        if (n + 16 <= p.N) {
          bf16 v[4];
          __builtin_memcpy(v, y, 8);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = static_cast<bf16>(static_cast<float>(v[e]) + o[e]);
          __builtin_memcpy(out, v, 8);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + 4 * g + e < p.N) out[e] = static_cast<bf16>(static_cast<float>(y[e]) + o[e]);
        }
      }
    }
  }
}

// ── which form ──────────────────────────────────────────────────────────────
// Two launches.  Up to 256 rows, which may all have adapters of their own, there are workgroups for each row, of which those
// that are not their adapter's first in 16 rows end at once.  More rows come as runs, as a rule, or as many requests' single
// tokens: tiles of rows, each with some workgroups that take its adapters in turn, and end if there are not as many.  Up to 512
// rows, where the rank is 16 or less: tiles of 16 rows with four; else of 32 (down: 64 past 1024) with three, past 512 rows two.
// us for 4096 -> 4096 of rank 16, 16 rows and four / 32 and three: 300 rows and 100 adapters 36 / 60 (a workgroup a row: 22),
// 500 rows of their own 46 / 74, runs of 100 rows, three 10.7 / 9.9 (17), five 13.2 / 10.8; past 512, 32 and two: 900 rows and 100
// adapters 63 / 118, but three runs of 300 14.9 / 12.9, five of 200, -> 11008, 23.2 / 17.6; of rank 64, 4096 -> 11008: five runs
// of 100 31 / 24.9, 500 rows and ten adapters 94 / 76.
// 2000 rows in five runs, rank 64, 4096 -> 11008: tiles of 16 / 32 / 64 for the columns 51.5 / 40.6 / 53.5, of 32 / 64 for the
// ranks 43.5 / 40.6 (800 rows: 24.5 / 26.9); 300 rows and 100 adapters, two / three / four workgroups to 32: 83 / 60 / 50, three
// runs of 300 12.6 / 15.5 / 16.0.
// down: 1024 k's or more to a split, since every range of columns sums all parts, and up to 512 workgroups or four splits (us
// for 512 k's / 1024: 64 rows and adapters of rank 64, 4096 -> 4096 21.7 / 19.2; 20 adapters, -> 11008 28.3 / 23.7; rank 16, 40
// adapters 11.6 / 10.8; two / four splits of two runs of 100 rows 10.6 / 9.3).
// up: ranges of columns for 768 workgroups, of which the idle ones cost little (us by 512 / 768 / 1024 / 2048 / 4096: rank 16, 64
// rows, 40 adapters, -> 11008 11.2 / 10.8 / 10.7 / 12.0 / 13.9; 200 rows, 100 adapters 25.6 / 25.4 / 27.9 / 28.4 / 27.8), or eight
// (two runs of 100 rows of rank 64: 4 / 6 / 10 34 / 31 / 26.5; 200 rows, 100 adapters 25.4 / 27.9 / 26.9); of many rows for 512
// (2000 rows of rank 64, -> 11008: 256 / 512 / 1024 / 2048 47.2 / 40.6 / 41.5 / 43.7; rank 16, 11008 -> 4096 29.4 / 28.3 / 30.2 / 30.1).
struct AdapterPlan {
  int rt = 1, down = 1, up = 1, slots = 0, splits = 1, chunk = 0, cols = 0;  // down, up: 16-row tiles of a workgroup
  bool one = false;  // one launch
  size_t bytes = 0;
};

static AdapterPlan adapter_plan(int64_t M, int64_t N, int64_t K, int64_t rank) {
  AdapterPlan pl;
  const bool many = M > 256;
  pl.rt = rank <= 16 ? 1 : rank <= 32 ? 2 : rank <= 64 ? 4 : 8;
  const bool small = !many || (pl.rt == 1 && M <= 512);  // tiles
  pl.down = small ? 1 : M > 1024 ? 4 : 2;
  pl.up = small ? 1 : 2;
  pl.slots = !many ? 0 : small ? 4 : M > 512 ? 2 : 3;
  const int64_t down = many ? cdiv(M, 16 * pl.down) : M, up = many ? cdiv(M, 16 * pl.up) : M;
  const int64_t splits = std::max<int64_t>(1, std::min(cdiv(K, 1024), std::max<int64_t>(small ? 4 : 1, cdiv(512, down))));
  pl.chunk = static_cast<int>(std::max<int64_t>(1, cdiv(cdiv(K, splits), 256)) * 256);
  pl.splits = static_cast<int>(cdiv(K, pl.chunk));
  const int64_t ranges = std::max<int64_t>(1, std::min(cdiv(N, 256), std::max<int64_t>(small ? 8 : 4, (many ? 512 : 768) / up)));
  pl.cols = static_cast<int>(cdiv(cdiv(N, ranges), 256) * 256);
  // One launch for few small products, each workgroup having a CU to itself: a row, rank 16, 1024 -> 4096: 5.6 us against
  // 6.4; 16 rows: 6.4 against 7.0; but every range of columns reads all of A: a row, 4096 -> 4096: 7.5 against 6.4 us
  // (2048 -> 2048: 6.9 both); more workgroups than CUs: 64 rows, 1024 -> 4096: 22.5 against 9.0 us.
  pl.one = 16 * pl.rt * K <= 16384 && M * cdiv(N, 256) <= 256;
  pl.bytes = pl.one ? 0 : static_cast<size_t>(pl.splits) * M * 16 * pl.rt * 4;
  return pl;
}

static dim3 adapter_grid(const AdapterPlan &pl, const AdapterArgs &p, int tiles, int64_t y) {
  return dim3(static_cast<unsigned>(pl.slots == 0 ? p.M : cdiv(p.M, 16 * tiles) * pl.slots), static_cast<unsigned>(y));
}
template <int RT>
static void launch_adapter(const AdapterPlan &pl, const AdapterArgs &p, hipStream_t s) {
  const dim3 down = adapter_grid(pl, p, pl.down, pl.splits), up = adapter_grid(pl, p, pl.up, cdiv(p.N, pl.cols));
  if (pl.down == 4) hipLaunchKernelGGL((adapter_down<RT, 4>), down, dim3(256), 0, s, p);
  else if (pl.down == 2) hipLaunchKernelGGL((adapter_down<RT, 2>), down, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((adapter_down<RT, 1>), down, dim3(256), 0, s, p);
  if (pl.up == 2) hipLaunchKernelGGL((adapter_up<RT, 2>), up, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((adapter_up<RT, 1>), up, dim3(256), 0, s, p);
}

}  // namespace teeny

using namespace teeny;

extern "C" {

teeny_status teeny_adapter_add(const void *x, const void *a, const void *b, const int32_t *adapters, const float *scale,
                               const void *y, void *out, int64_t M, int64_t N, int64_t K, int64_t rank,
                               int64_t num_adapters, int64_t x_stride, int64_t y_stride, int64_t out_stride,
                               teeny_stream stream) {
  const char *nm = "adapter_add";
  TEENY_REQUIRE(M >= 0 && N >= 0 && K >= 0 && rank >= 0 && num_adapters >= 0, TEENY_ERR_SHAPE_MISMATCH,
                "adapter_add: negative size");
  TEENY_REQUIRE(M <= 1 << 24 && N <= 1 << 24 && K <= 1 << 22 && num_adapters <= 1 << 24, TEENY_ERR_SHAPE_MISMATCH,
                "adapter_add: M, N or num_adapters exceed 2^24, or K 2^22");
  TEENY_REQUIRE(N * rank < 1 << 30, TEENY_ERR_SHAPE_MISMATCH, "adapter_add: N * rank must be below 2^30");
  TEENY_REQUIRE(K % 8 == 0, TEENY_ERR_SHAPE_MISMATCH, "adapter_add: K must be a multiple of 8");
  TEENY_REQUIRE(rank % 8 == 0 && rank <= 128, TEENY_ERR_UNSUPPORTED, "adapter_add: rank must be a multiple of 8 up to 128");
  if (M == 0 || N == 0) return TEENY_OK;
  TEENY_REQUIRE(adapters != nullptr && y != nullptr && out != nullptr, TEENY_ERR_NULL_POINTER, "adapter_add: adapters/y/out");
  TEENY_REQUIRE(y_stride >= N && out_stride >= N && y_stride <= 1 << 24 && out_stride <= 1 << 24, TEENY_ERR_SHAPE_MISMATCH,
                "adapter_add: row strides below N or above 2^24");
  TEENY_REQUIRE(y != out || y_stride == out_stride, TEENY_ERR_INVALID_ARGUMENT,
                "adapter_add: out can be y only with the same row stride");
  if (rank == 0 || K == 0) num_adapters = 0;
  TEENY_REQUIRE(num_adapters == 0 || (x != nullptr && a != nullptr && b != nullptr), TEENY_ERR_NULL_POINTER,
                "adapter_add: x/a/b");
  TEENY_REQUIRE(num_adapters == 0 || (x_stride >= K && x_stride <= 1 << 24), TEENY_ERR_SHAPE_MISMATCH,
                "adapter_add: x's row stride below K or above 2^24");
  TEENY_REQUIRE(num_adapters == 0 || (aligned(x, 16) && aligned(a, 16) && aligned(b, 16) && x_stride % 8 == 0),
                TEENY_ERR_MISALIGNED, "adapter_add: 16-byte aligned x, a, b and x's row stride");
  AdapterArgs p{static_cast<const bf16 *>(x), static_cast<const bf16 *>(a), static_cast<const bf16 *>(b), adapters, scale,
                static_cast<const bf16 *>(y), static_cast<bf16 *>(out), x_stride, y_stride, out_stride,
                static_cast<int>(M), static_cast<int>(N), static_cast<int>(K), static_cast<int>(rank),
                static_cast<int>(num_adapters), 0, nullptr, 1, 0, 0};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const AdapterPlan pl = adapter_plan(M, N, K, rank);
  const Scratch scr = stream_scratch(s);
  if (num_adapters > 0 && !pl.one && scr.ptr != nullptr && scr.bytes >= pl.bytes) {
    p.part = static_cast<float *>(scr.ptr);
    p.cols = pl.cols;
    p.splits = pl.splits;
    p.chunk = pl.chunk;
    p.slots = pl.slots;
    switch (pl.rt) {
      case 1: launch_adapter<1>(pl, p, s); break;
      case 2: launch_adapter<2>(pl, p, s); break;
      case 4: launch_adapter<4>(pl, p, s); break;
      default: launch_adapter<8>(pl, p, s); break;
    }
    return after_launch(nm, s);
  }
  p.slots = M <= 256 ? 0 : 1;
  p.cols = static_cast<int>(cdiv(cdiv(N, std::max<int64_t>(1, 512 / cdiv(M, 16))), 256) * 256);
  const dim3 grid(static_cast<unsigned>(p.slots == 0 ? M : cdiv(M, 16)), static_cast<unsigned>(cdiv(N, p.cols)));
  switch (pl.rt) {
    case 1: hipLaunchKernelGGL(adapter_one<1>, grid, dim3(1024), 0, s, p); break;
    case 2: hipLaunchKernelGGL(adapter_one<2>, grid, dim3(1024), 0, s, p); break;
    case 4: hipLaunchKernelGGL(adapter_one<4>, grid, dim3(1024), 0, s, p); break;
    default: hipLaunchKernelGGL(adapter_one<8>, grid, dim3(1024), 0, s, p); break;
  }
  return after_launch(nm, s);
}

teeny_status teeny_adapter_add_workspace_size(int64_t M, int64_t N, int64_t K, int64_t rank, size_t *bytes) {
  TEENY_REQUIRE(bytes != nullptr, TEENY_ERR_NULL_POINTER, "adapter_add_workspace_size: bytes");
  *bytes = 0;
  TEENY_REQUIRE(M >= 0 && N >= 0 && K >= 0 && rank >= 0 && M <= 1 << 24 && N <= 1 << 24 && K <= 1 << 22,
                TEENY_ERR_SHAPE_MISMATCH, "adapter_add_workspace_size: sizes out of range");
  TEENY_REQUIRE(rank % 8 == 0 && rank <= 128, TEENY_ERR_UNSUPPORTED,
                "adapter_add_workspace_size: rank must be a multiple of 8 up to 128");
  if (M > 0 && N > 0 && K > 0 && rank > 0) *bytes = adapter_plan(M, N, K, rank).bytes;
  return TEENY_OK;
}

}  // extern "C"
