// Low-rank adapters of many requests beside a projection that they share:
//
//   out[m] = y[m] + scale[a] B[a] (A[a] x[m]),  a = adapters[m] (none: out[m] = y[m])
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
  int M, N, K, rank, adapters, vec;  // vec: rows of y and out are aligned for eight numbers
  int cols;                          // output columns of a workgroup
  float *part;                       // [splits][M][RP] products of the ranks, RP: the rank in whole tiles of 16
  int splits, chunk, by_row;         // chunk: k's of a split; by_row: workgroups by rows, not by tiles of them
};

__device__ __forceinline__ f32x4 mfma_16x16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ bf16x8 load8(const bf16 *p, bool there) {
  const u32x4 v = there ? *reinterpret_cast<const u32x4 *>(p) : u32x4{0u, 0u, 0u, 0u};
  return __builtin_bit_cast(bf16x8, v);
}

// 16 numbers of a row of the output from those of y and of the adapter.
__device__ __forceinline__ void adapter_store(const AdapterArgs &p, int m, int n, const f32x4 (&add)[4]) {
  const bf16 *y = p.y + m * p.y_stride + n;
  bf16 *out = p.out + m * p.out_stride + n;
  if (p.vec && n + 16 <= p.N) {
    bf16x8 v[2] = {*reinterpret_cast<const bf16x8 *>(y), *reinterpret_cast<const bf16x8 *>(y + 8)};
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i >> 3][i & 7] = static_cast<bf16>(static_cast<float>(v[i >> 3][i & 7]) + add[i >> 2][i & 3]);
    *reinterpret_cast<bf16x8 *>(out) = v[0];
    *reinterpret_cast<bf16x8 *>(out + 8) = v[1];
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (n + i < p.N) out[i] = static_cast<bf16>(static_cast<float>(y[i]) + add[i >> 2][i & 3]);
  }
}

// The rows of one adapter among 16 MT rows: lane l's row l.
template <int MT>
struct AdapterRows {
  int m0, id;     // the first row; the lane's adapter (-1: none, -2: no row)
  uint64_t left;  // rows that are still to be taken up, by the first of each adapter's
  __device__ __forceinline__ AdapterRows(const AdapterArgs &p, int block) {
    const int lane = threadIdx.x & 63;
    m0 = p.by_row ? block & ~(16 * MT - 1) : block * 16 * MT;
    id = -2;
    if (lane < 16 * MT && m0 + lane < p.M) {
      id = p.ids[m0 + lane];
      if (id < 0 || id >= p.adapters) id = -1;
    }
    left = __ballot(id >= -1);
    if (p.by_row) {
      // the workgroup of an adapter's first row takes all of its rows
      const int at = block - m0;
      const uint64_t same = __ballot(id == __builtin_amdgcn_readlane(id, at));
      left = __builtin_ctzll(same) == at ? same : 0;
    }
  }
  // the next adapter; its rows
  __device__ __forceinline__ int next(uint64_t &rows) {
    const int a = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
    rows = __ballot(id == a);
    left &= ~rows;
    return a;
  }
};

// part[split] = A[a] x over the split's k's.  Four waves share them out in turn, 64 at
// a time, and meet in LDS.  Rows of other adapters are multiplied too and not
// written; rows of A past the rank repeat the last one and are not read again.
template <int RT, int MT>
__global__ __launch_bounds__(256) void adapter_down(AdapterArgs p) {
  constexpr int U = RT * MT >= 8 ? 1 : RT * MT >= 4 ? 2 : 4, RP = 16 * RT;
  __shared__ __attribute__((aligned(16))) float sum[4][16 * MT][RP + 4];
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, c = lane & 15, g = lane >> 4;
  AdapterRows<MT> rows(p, blockIdx.x);
  const int kb = blockIdx.y * p.chunk, ke = min(p.K, kb + p.chunk);
  const bf16 *x[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) x[t] = p.x + min(rows.m0 + 16 * t + c, p.M - 1) * p.x_stride + 8 * g;
  while (rows.left != 0) {
    uint64_t mine;
    const int a = rows.next(mine);
    if (a < 0) continue;
    const bf16 *ar[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) ar[t] = p.a + (static_cast<int64_t>(a) * p.rank + min(16 * t + c, p.rank - 1)) * p.K + 8 * g;
    f32x4 acc[RT][MT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[r][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    int k = kb + 64 * w;
    for (; k + 256 * (U - 1) + 64 <= ke; k += 256 * U) {
      bf16x8 xf[U][2][MT], af[U][2][RT];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int at = k + 256 * u + 32 * h;
#pragma unroll
          for (int r = 0; r < RT; ++r) af[u][h][r] = *reinterpret_cast<const bf16x8 *>(ar[r] + at);
#pragma unroll
          for (int t = 0; t < MT; ++t) xf[u][h][t] = *reinterpret_cast<const bf16x8 *>(x[t] + at);
        }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[r][t] = mfma_16x16(af[u][h][r], xf[u][h][t], acc[r][t]);
    }
    for (; k < ke; k += 256)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = k + 32 * h;
        const bool in = at + 8 * g < ke;
        bf16x8 xf[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) xf[t] = load8(x[t] + at, in);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const bf16x8 af = load8(ar[r] + at, in);
#pragma unroll
          for (int t = 0; t < MT; ++t) acc[r][t] = mfma_16x16(af, xf[t], acc[r][t]);
        }
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

// out = y + B[a] (scale part).  A wave takes 64 columns a time, 16 to each lane group:
// 16 consecutive numbers of a row of the output are one lane's.  The ranks'
// products are two bf16 parts of an fp32 number; at a rank of 16 or less both are
// the k's of one product.
template <int RT, int MT>
__global__ __launch_bounds__(256) void adapter_up(AdapterArgs p) {
  constexpr int RP = 16 * RT, KS = RT == 1 ? 1 : RT / 2, LH = (RT == 1 ? 32 : RP) + 8, PARTS = RT == 1 ? 1 : 2;
  __shared__ __attribute__((aligned(16))) bf16 hs[PARTS][16 * MT][LH];
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, c = lane & 15, g = lane >> 4;
  AdapterRows<MT> rows(p, blockIdx.x);
  const int n0 = blockIdx.y * p.cols, n1 = min(p.N, n0 + p.cols);
  while (rows.left != 0) {
    uint64_t mine;
    const int a = rows.next(mine);
    if (a < 0) {
      if (p.out == p.y) continue;
      const f32x4 zero[4] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f},
                             f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
      for (int n = n0 + 64 * w + 16 * g; n < n1; n += 256)
#pragma unroll
        for (int t = 0; t < MT; ++t)
          if ((mine >> (16 * t + c)) & 1) adapter_store(p, rows.m0 + 16 * t + c, n, zero);
      continue;
    }
    const float scale = p.scale != nullptr ? p.scale[a] : 1.0f;
    __syncthreads();  // the last adapter's products have been read
    for (int i = tid; i < 16 * MT * RP; i += 256) {
      const int m = i / RP, r = i - m * RP;
      float h = 0.0f;
      if (r < p.rank && ((mine >> m) & 1)) {
        const float *at = p.part + static_cast<int64_t>(rows.m0 + m) * RP + r;
        for (int s = 0; s < p.splits; ++s) h += at[static_cast<int64_t>(s) * p.M * RP];
        h *= scale;
      }
      const bf16 hi = static_cast<bf16>(h);
      const bf16 lo = fabsf(static_cast<float>(hi)) < INFINITY ? static_cast<bf16>(h - static_cast<float>(hi)) : static_cast<bf16>(0.0f);
      hs[0][m][r] = hi;
      if constexpr (RT == 1) hs[0][m][16 + r] = lo;
      else hs[PARTS - 1][m][r] = lo;
    }
    __syncthreads();
    const int r0 = RT == 1 ? 8 * (g & 1) : 8 * g;
    const bf16 *b = p.b + static_cast<int64_t>(a) * p.N * p.rank;
    for (int n = n0 + 64 * w; n < n1; n += 256) {
      bf16x8 bf[4][KS];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bf16 *at = b + static_cast<int64_t>(min(n + 16 * (c >> 2) + 4 * j + (c & 3), p.N - 1)) * p.rank + r0;
#pragma unroll
        for (int k = 0; k < KS; ++k) bf[j][k] = load8(at + 32 * k, r0 + 32 * k < p.rank);
      }
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        f32x4 o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          o[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int s = 0; s < PARTS; ++s)
#pragma unroll
            for (int k = 0; k < KS; ++k)
              o[j] = mfma_16x16(bf[j][k], *reinterpret_cast<const bf16x8 *>(&hs[s][16 * t + c][32 * k + 8 * g]), o[j]);
        }
        if ((mine >> (16 * t + c)) & 1) adapter_store(p, rows.m0 + 16 * t + c, n + 16 * g, o);
      }
    }
  }
}

// One workgroup for 16 rows and a range of columns, without scratch: the ranks'
// products for these rows are summed in LDS, once for each range of columns.
template <int RT>  // 16-row tiles of the rank
__global__ __launch_bounds__(256) void adapter_one(AdapterArgs p) {
  constexpr int LR = 16 * RT + 4;
  __shared__ __attribute__((aligned(16))) float part[4][16][LR];
  __shared__ __attribute__((aligned(16))) bf16 hs[2][16][16 * RT + 24];  // [hi, lo]; k past the rank's tiles read as zeros
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int m0 = blockIdx.x * 16, n0 = blockIdx.y * p.cols, n1 = min(p.N, n0 + p.cols);
  const int row = min(m0 + c, p.M - 1);
  int id = m0 + c < p.M ? p.ids[row] : -1;
  if (id < 0 || id >= p.adapters) id = -1;
  const bool here = m0 + c < p.M;
  const f32x4 zero[4] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f},
                         f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
  // rows of no adapter
  for (int n = n0 + 64 * w + 16 * g; n < n1; n += 256)
    if (here && id < 0) adapter_store(p, row, n, zero);
  uint64_t left = __ballot(id >= 0) & 0xffffu;
  while (left != 0) {
    const int a = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
    const bool mine = id == a;
    left &= ~__ballot(mine);
    f32x4 acc[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const bf16 *x = p.x + row * p.x_stride;
    for (int k = 32 * w; k < p.K; k += 128) {
      const bool in = k + 8 * g < p.K;
      const bf16x8 xf = load8(x + k + 8 * g, in && mine);
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const int r = 16 * t + c;
        acc[t] = mfma_16x16(load8(p.a + (static_cast<int64_t>(a) * p.rank + r) * p.K + k + 8 * g, in && r < p.rank), xf, acc[t]);
      }
    }
    __syncthreads();  // the last round's products have been read
#pragma unroll
    for (int t = 0; t < RT; ++t) *reinterpret_cast<f32x4 *>(&part[w][c][16 * t + 4 * g]) = acc[t];
    __syncthreads();
    const float scale = p.scale != nullptr ? p.scale[a] : 1.0f;
    for (int i = tid; i < 16 * (16 * RT + 16); i += 256) {
      const int m = i / (16 * RT + 16), r = i - m * (16 * RT + 16);
      const float h = r < 16 * RT ? scale * (part[0][m][r] + part[1][m][r] + part[2][m][r] + part[3][m][r]) : 0.0f;
      const bf16 hi = static_cast<bf16>(h);
      hs[0][m][r] = hi;
      hs[1][m][r] = fabsf(static_cast<float>(hi)) < INFINITY ? static_cast<bf16>(h - static_cast<float>(hi)) : static_cast<bf16>(0.0f);
    }
    __syncthreads();
    for (int n = n0 + 64 * w; n < n1; n += 256) {
      f32x4 o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        o[j] = zero[j];
        const int col = n + 16 * (c >> 2) + 4 * j + (c & 3);
#pragma unroll
        for (int k = 0; k < 16 * RT; k += 32) {
          const bf16x8 bf = load8(p.b + (static_cast<int64_t>(a) * p.N + col) * p.rank + k + 8 * g, col < p.N && k + 8 * g < p.rank);
#pragma unroll
          for (int s = 0; s < 2; ++s) o[j] = mfma_16x16(bf, *reinterpret_cast<const bf16x8 *>(&hs[s][c][k + 8 * g]), o[j]);
        }
      }
      if (mine && here) adapter_store(p, row, n + 16 * g, o);
    }
  }
}

// ── which form ──────────────────────────────────────────────────────────────
struct AdapterPlan {
  int rt = 1, mt = 1, splits = 1, chunk = 0, cols = 0;
  bool by_row = false;
  size_t bytes = 0;
};

static AdapterPlan adapter_plan(int64_t M, int64_t N, int64_t K, int64_t rank) {
  AdapterPlan pl;
  pl.rt = rank <= 16 ? 1 : rank <= 32 ? 2 : rank <= 64 ? 4 : 8;
  pl.by_row = M <= 256;
  pl.mt = pl.by_row ? 1 : 2;
  const int64_t units = pl.by_row ? M : cdiv(M, 16 * pl.mt);
  const int64_t splits = std::max<int64_t>(1, std::min(cdiv(K, 1024), cdiv(512, units)));
  pl.chunk = static_cast<int>(std::max<int64_t>(1, cdiv(cdiv(K, splits), 256)) * 256);
  pl.splits = static_cast<int>(cdiv(K, pl.chunk));
  const int64_t ranges = std::max<int64_t>(1, std::min(cdiv(N, 1024), cdiv(1024, units)));
  pl.cols = static_cast<int>(cdiv(cdiv(N, ranges), 256) * 256);
  pl.bytes = static_cast<size_t>(pl.splits) * M * 16 * pl.rt * 4;
  return pl;
}

template <int RT, int MT>
static void launch_adapter(const AdapterPlan &pl, const AdapterArgs &p, hipStream_t s) {
  const unsigned units = static_cast<unsigned>(pl.by_row ? p.M : cdiv(p.M, 16 * MT));
  hipLaunchKernelGGL((adapter_down<RT, MT>), dim3(units, static_cast<unsigned>(pl.splits)), dim3(256), 0, s, p);
  hipLaunchKernelGGL((adapter_up<RT, MT>), dim3(units, static_cast<unsigned>(cdiv(p.N, pl.cols))), dim3(256), 0, s, p);
}
template <int RT>
static void launch_adapter(const AdapterPlan &pl, const AdapterArgs &p, hipStream_t s) {
  if (pl.mt == 2) launch_adapter<RT, 2>(pl, p, s);
  else launch_adapter<RT, 1>(pl, p, s);
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
  TEENY_REQUIRE(M <= 1 << 24 && N <= 1 << 24 && K <= 1 << 24 && num_adapters <= 1 << 24, TEENY_ERR_SHAPE_MISMATCH,
                "adapter_add: M, N, K or num_adapters exceed 2^24");
  TEENY_REQUIRE(K % 8 == 0, TEENY_ERR_SHAPE_MISMATCH, "adapter_add: K must be a multiple of 8");
  TEENY_REQUIRE(rank % 8 == 0 && rank <= 128, TEENY_ERR_UNSUPPORTED, "adapter_add: rank must be a multiple of 8 up to 128");
  if (M == 0 || N == 0) return TEENY_OK;
  TEENY_REQUIRE(adapters != nullptr && y != nullptr && out != nullptr, TEENY_ERR_NULL_POINTER, "adapter_add: adapters/y/out");
  TEENY_REQUIRE(y_stride >= N && out_stride >= N, TEENY_ERR_SHAPE_MISMATCH, "adapter_add: row strides below N");
  TEENY_REQUIRE(y != out || y_stride == out_stride, TEENY_ERR_INVALID_ARGUMENT,
                "adapter_add: out can be y only with the same row stride");
  if (rank == 0 || K == 0) num_adapters = 0;
  TEENY_REQUIRE(num_adapters == 0 || (x != nullptr && a != nullptr && b != nullptr), TEENY_ERR_NULL_POINTER,
                "adapter_add: x/a/b");
  TEENY_REQUIRE(num_adapters == 0 || x_stride >= K, TEENY_ERR_SHAPE_MISMATCH, "adapter_add: row stride below K");
  TEENY_REQUIRE(num_adapters == 0 || (aligned(x, 16) && aligned(a, 16) && aligned(b, 16) && x_stride % 8 == 0),
                TEENY_ERR_MISALIGNED, "adapter_add: 16-byte aligned x, a, b and x's row stride");
  AdapterArgs p{static_cast<const bf16 *>(x), static_cast<const bf16 *>(a), static_cast<const bf16 *>(b), adapters, scale,
                static_cast<const bf16 *>(y), static_cast<bf16 *>(out), x_stride, y_stride, out_stride,
                static_cast<int>(M), static_cast<int>(N), static_cast<int>(K), static_cast<int>(rank),
                static_cast<int>(num_adapters),
                aligned(y, 16) && aligned(out, 16) && y_stride % 8 == 0 && out_stride % 8 == 0, 0, nullptr, 1, 0, 0};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const AdapterPlan pl = adapter_plan(M, N, K, rank);
  const Scratch scr = stream_scratch(s);
  if (num_adapters > 0 && scr.ptr != nullptr && scr.bytes >= pl.bytes) {
    p.part = static_cast<float *>(scr.ptr);
    p.cols = pl.cols;
    p.splits = pl.splits;
    p.chunk = pl.chunk;
    p.by_row = pl.by_row;
    switch (pl.rt) {
      case 1: launch_adapter<1>(pl, p, s); break;
      case 2: launch_adapter<2>(pl, p, s); break;
      case 4: launch_adapter<4>(pl, p, s); break;
      default: launch_adapter<8>(pl, p, s); break;
    }
    return after_launch(nm, s);
  }
  const int64_t tiles = cdiv(M, 16), ranges = std::min<int64_t>(cdiv(N, 256), cdiv(512, tiles));
  p.cols = static_cast<int>(cdiv(cdiv(N, ranges), 256) * 256);
  const dim3 grid(static_cast<unsigned>(tiles), static_cast<unsigned>(cdiv(N, p.cols)));
  switch ((rank + 15) / 16) {
    case 0:
    case 1: hipLaunchKernelGGL(adapter_one<1>, grid, dim3(256), 0, s, p); break;
    case 2: hipLaunchKernelGGL(adapter_one<2>, grid, dim3(256), 0, s, p); break;
    case 3:
    case 4: hipLaunchKernelGGL(adapter_one<4>, grid, dim3(256), 0, s, p); break;
    default: hipLaunchKernelGGL(adapter_one<8>, grid, dim3(256), 0, s, p); break;
  }
  return after_launch(nm, s);
}

teeny_status teeny_adapter_add_workspace_size(int64_t M, int64_t N, int64_t K, int64_t rank, size_t *bytes) {
  TEENY_REQUIRE(bytes != nullptr, TEENY_ERR_NULL_POINTER, "adapter_add_workspace_size: bytes");
  *bytes = 0;
  TEENY_REQUIRE(M >= 0 && N >= 0 && K >= 0 && rank >= 0 && M <= 1 << 24 && N <= 1 << 24 && K <= 1 << 24,
                TEENY_ERR_SHAPE_MISMATCH, "adapter_add_workspace_size: sizes out of range");
  TEENY_REQUIRE(rank % 8 == 0 && rank <= 128, TEENY_ERR_UNSUPPORTED,
                "adapter_add_workspace_size: rank must be a multiple of 8 up to 128");
  if (M > 0 && N > 0 && K > 0 && rank > 0) *bytes = adapter_plan(M, N, K, rank).bytes;
  return TEENY_OK;
}

}  // extern "C"
