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
  int M, N, K, rank, adapters, vec;  // vec: rows of y and out are aligned for four numbers
  int cols;                          // output columns of a workgroup
};

__device__ __forceinline__ f32x4 mfma_16x16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ bf16x8 load8(const bf16 *p, bool there) {
  const u32x4 v = there ? *reinterpret_cast<const u32x4 *>(p) : u32x4{0u, 0u, 0u, 0u};
  return __builtin_bit_cast(bf16x8, v);
}

// Four numbers of a row of the output from those of y and of the adapter.
__device__ __forceinline__ void adapter_store(const AdapterArgs &p, int m, int n, f32x4 add) {
  const bf16 *y = p.y + m * p.y_stride + n;
  bf16 *out = p.out + m * p.out_stride + n;
  if (p.vec && n + 4 <= p.N) {
    bf16x4 v = *reinterpret_cast<const bf16x4 *>(y);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = static_cast<bf16>(static_cast<float>(v[i]) + add[i]);
    *reinterpret_cast<bf16x4 *>(out) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < p.N) out[i] = static_cast<bf16>(static_cast<float>(y[i]) + add[i]);
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
  // rows of no adapter
  for (int n = n0 + 16 * w + 4 * g; n < n1; n += 64)
    if (here && id < 0) adapter_store(p, row, n, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
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
    for (int n = n0 + 16 * w; n < n1; n += 64) {
      f32x4 o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < 16 * RT; k += 32) {
        const bf16x8 bf = load8(p.b + (static_cast<int64_t>(a) * p.N + n + c) * p.rank + k + 8 * g, n + c < p.N && k + 8 * g < p.rank);
#pragma unroll
        for (int s = 0; s < 2; ++s) o = mfma_16x16(bf, *reinterpret_cast<const bf16x8 *>(&hs[s][c][k + 8 * g]), o);
      }
      if (mine && here) adapter_store(p, row, n + 4 * g, o);
    }
  }
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
                aligned(y, 8) && aligned(out, 8) && y_stride % 4 == 0 && out_stride % 4 == 0, 0};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t tiles = cdiv(M, 16), ranges = std::min<int64_t>(cdiv(N, 64), cdiv(512, tiles));
  p.cols = static_cast<int>(cdiv(cdiv(N, ranges), 64) * 64);
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

}  // extern "C"
