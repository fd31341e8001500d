// The 4-bit paged K/V cache: a step's tokens rotated and appended.
//
// No counterpart in the reference, whose attention reads dense K and V and rotates
// nothing (kernels/teeny-kernels/src/nn/attention/flash_attn2.rs:18-21).  Each
// token's head is held in groups of 64 numbers with a scale of their own, so a
// token never changes another's codes (kv_cache.hip's pages have one scale, which
// can grow).  Of a group's numbers m is the one of largest magnitude (of two, the
// positive one): s = -m / 8 with five significant bits, code = rint(x / s) in
// -8..7.  The sign lets the largest take the code -8, which symmetric codes never
// use (normal values: rms error 0.095 of the standard deviation, 0.108 with m / 7);
// five bits times a code are a bf16 number, so that attention can multiply in
// bf16 without another rounding (it costs 0.2 % of the error).
//
// Layouts (chosen for kv4_attn.hip's operands): K [pages, heads, page_size, D / 2]
// bytes, a token's word 2 (D / 64) g + 2 G + j holds group G's numbers 16 g + 8 j +
// 0..7; V [pages, heads, page_size / 16, D, 8] bytes, word h of a d holds tokens 8 h
// + 0..7 of the 16; nibbles as w4_nibble; scales bf16 [pages, heads, page_size, D / 64].
#include "kv4.hpp"

namespace teeny {

struct Kv4AppendArgs {
  const bf16 *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;
  const int32_t *positions, *slots;
  const float *inv_freq;
  bf16 *q_out;
  int8_t *kc, *vc;
  bf16 *ks, *vs;
  int tokens, q_heads, kv_heads, limit, shift;  // limit: slots of the cache
  int half, interleaved;                        // rotated pairs of a head
  int per, rows_grid;                           // tokens per workgroup of rows, workgroups of rows
  int share;                                    // workgroups to 64 tokens' V of a head
};

// m / -8 with five significant bits, to nearest even; key: magnitude bits and, lowest, whether positive.  Below 2^-90
// zero (every code is 0), and NaN where the group holds an infinity or NaN.
__device__ __forceinline__ float kv4_scale(uint32_t key) {
  const uint32_t mag = key >> 1;
  if (mag >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  if (mag < (37u << 23)) return 0.0f;  // 2^-90
  const uint32_t eighth = (mag - (3u << 23)) | (key << 31);  // the positive one takes the sign
  return __uint_as_float((eighth + 0x3ffffu + ((eighth >> 19) & 1u)) & 0xfff80000u);
}
// 1 / s of such a scale, correctly rounded (0 for 0): one Newton step from the approximation, checked for each of the 16
// significands.
__device__ __forceinline__ float kv4_inverse(float s) {
  const float r = __builtin_amdgcn_rcpf(s);
  return s == 0.0f ? 0.0f : __builtin_fmaf(__builtin_fmaf(-s, r, 1.0f), r, r);
}
// Code + 8, in the low four bits: rint of the quotient.  x inv is corrected by the exact remainder.  Once suffices where
// the quotient of an 8-bit by a 5-bit significand is either a half exactly or far from one; twice gives the fp32 quotient
// of any x (Markstein, 1990).  Adding 1.5 * 2^23 rounds to an integer and leaves it in the low bits.
template <int TIMES>
__device__ __forceinline__ uint32_t kv4_code(float x, float s, float inv) {
  float t = x * inv;
#pragma unroll
  for (int i = 0; i < TIMES; ++i) t = __builtin_fmaf(__builtin_fmaf(-t, s, x), inv, t);
  return __float_as_uint(fminf(t, 7.0f) + 12582920.0f) & 15u;
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, true));
}
// Maximum over 8 lanes, in each of them: quad_perm [1, 0, 3, 2] and [2, 3, 0, 1], row_half_mirror.
template <typename F>
__device__ __forceinline__ uint32_t over8(uint32_t v, F f) {
  v = f(v, dpp<0xb1>(v));
  v = f(v, dpp<0x4e>(v));
  return f(v, dpp<0x141>(v));
}

// Rows of q and k: D / 8 lanes a row, eight numbers each and their partners.  The angles' cosines and sines are taken
// once per token, in 64 bits, as are the rotated keys: a code that falls on the other side of a half would be a whole
// step off.  Queries, which are rounded to bf16 next, take fp32 cosines, sines and products: within 2^-22 of the pair's
// larger number.  Keys are first, with the loads of the next rows of queries ahead of the work of this one's.  Bound by
// memory where there are many tokens: 8000 of 32 and 8 heads of 128 move 173 MB in 39 us, 4.4 TB/s (43 to 45 in a graph
// whose calls take other inputs each).
template <int D>
__device__ __forceinline__ void kv4_rows(const Kv4AppendArgs &p, int block) {
  constexpr int LPR = D / 8, NG = D / 64, PASS = 256 / LPR, U = 4;
  __shared__ double2 turn64[4][64];
  __shared__ float2 turn32[4][64];
  __shared__ int at_pos[4], at_slot[4];
  const int tid = threadIdx.x, t0 = block * p.per, n = min(p.per, p.tokens - t0);
  if (tid < n) {
    const int pos = p.positions[t0 + tid], slot = p.kv_heads > 0 ? p.slots[t0 + tid] : -1;
    at_pos[tid] = pos;
    at_slot[tid] = pos >= 0 && slot < p.limit ? slot : -1;
  }
  if ((tid >> 6) < n && (tid & 63) < p.half) {
    const int pos = p.positions[t0 + (tid >> 6)];
    const double angle = static_cast<double>(pos) * static_cast<double>(p.inv_freq[tid & 63]);
    double2 cs;
    sincos(angle, &cs.y, &cs.x);
    turn64[tid >> 6][tid & 63] = cs;
    turn32[tid >> 6][tid & 63] = float2{static_cast<float>(cs.x), static_cast<float>(cs.y)};
  }
  const int m = tid % LPR, d0 = 8 * m;
  const bool turned = d0 < 2 * p.half, upper = !p.interleaved && d0 >= p.half;
  const int f0 = p.interleaved ? d0 / 2 : upper ? d0 - p.half : d0;  // the lane's first angle
  const int other = p.interleaved || !turned ? 0 : upper ? -p.half : p.half;
  // the first two rows of k are on their way while the angles are worked out
  auto k_row = [&](int row) {
    const int i = row / p.kv_heads, head = row - i * p.kv_heads;
    return p.k + (t0 + i) * p.k_stride + head * D + d0;
  };
  const int k_rows = n * p.kv_heads, k_first = tid / LPR;
  bf16x8 ka[2], kb[2];
  if (k_rows > 0)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const bf16 *src = k_row(min(k_first + u * PASS, k_rows - 1));
      ka[u] = *reinterpret_cast<const bf16x8 *>(src);
      kb[u] = *reinterpret_cast<const bf16x8 *>(src + other);
    }
  __syncthreads();
  for (int row = k_first, u = 0; row < k_rows; row += PASS, ++u) {
    const int i = row / p.kv_heads, head = row - i * p.kv_heads, slot = at_slot[i];
    bf16x8 a = ka[0], b = kb[0];
    ka[0] = ka[1], kb[0] = kb[1];
    if (u >= 2) {
      const bf16 *src = k_row(row);
      a = *reinterpret_cast<const bf16x8 *>(src);
      b = *reinterpret_cast<const bf16x8 *>(src + other);
    }
    if (slot < 0) continue;
    float y[8];
    const double2 *turn = turn64[i] + f0;
    if (!turned) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = static_cast<float>(a[e]);
    } else if (p.interleaved) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const double2 cs = turn[e];
        const double x1 = static_cast<float>(a[2 * e]), x2 = static_cast<float>(a[2 * e + 1]);
        y[2 * e] = static_cast<float>(__builtin_fma(x1, cs.x, -x2 * cs.y));
        y[2 * e + 1] = static_cast<float>(__builtin_fma(x2, cs.x, x1 * cs.y));
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double2 cs = turn[e];
        const double x = static_cast<float>(a[e]), o = static_cast<float>(b[e]);
        y[e] = static_cast<float>(__builtin_fma(x, cs.x, upper ? o * cs.y : -o * cs.y));
      }
    }
    uint32_t key = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t u = __float_as_uint(y[e]);
      key = max(key, (u << 1) | (~u >> 31));
    }
    key = over8(key, [](uint32_t x, uint32_t z) { return max(x, z); });
    const float s = kv4_scale(key), inv = kv4_inverse(s);
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) word |= kv4_code<2>(y[e], s, inv) << (4 * w4_nibble(e));
    if (!(s == s)) word = 0x88888888u;
    const int64_t token = ((static_cast<int64_t>(slot >> p.shift) * p.kv_heads + head) << p.shift) + (slot & ((1 << p.shift) - 1));
    *reinterpret_cast<uint32_t *>(p.kc + token * (D / 2) + 4 * (NG * (m & 6) + 2 * (m >> 3) + (m & 1))) = word;
    if ((m & 7) == 0) p.ks[token * NG + (m >> 3)] = static_cast<bf16>(s);
  }
  const int q_rows = n * p.q_heads;
  for (int row0 = tid / LPR; row0 < q_rows; row0 += U * PASS) {  // U rows' loads at once
    bf16x8 a[U], b[U];
    int at[U], head[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int row = min(row0 + u * PASS, q_rows - 1);
      at[u] = row / p.q_heads;
      head[u] = row - at[u] * p.q_heads;
      const bf16 *src = p.q + (t0 + at[u]) * p.q_stride + head[u] * D + d0;
      a[u] = *reinterpret_cast<const bf16x8 *>(src);
      b[u] = *reinterpret_cast<const bf16x8 *>(src + other);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (row0 + u * PASS >= q_rows || at_pos[at[u]] < 0) continue;
      bf16x8 y = a[u];
      if (turned) {
        const float2 *turn = turn32[at[u]] + f0;
        if (p.interleaved) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 cs = turn[e];
            const float x1 = static_cast<float>(a[u][2 * e]), x2 = static_cast<float>(a[u][2 * e + 1]);
            y[2 * e] = static_cast<bf16>(__builtin_fmaf(x1, cs.x, -x2 * cs.y));
            y[2 * e + 1] = static_cast<bf16>(__builtin_fmaf(x2, cs.x, x1 * cs.y));
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 cs = turn[e];
            const float x = static_cast<float>(a[u][e]), o = static_cast<float>(b[u][e]);
            y[e] = static_cast<bf16>(__builtin_fmaf(x, cs.x, upper ? o * cs.y : -o * cs.y));
          }
        }
      }
      *reinterpret_cast<bf16x8 *>(p.q_out + (static_cast<int64_t>(t0 + at[u]) * p.q_heads + head[u]) * D + d0) = y;
    }
  }
}

// V: the new tokens of 16 slots that one word pair of each d holds are a run of
// consecutive slots.  A wave takes a run and a head, D / 64 d's a lane, and writes
// whole words, with the nibbles of other tokens as they were.  Lane c of each 16
// has token c's scale.
template <int D>
__device__ __forceinline__ void kv4_values(const Kv4AppendArgs &p, int block) {
  constexpr int DPL = D / 64, NG = D / 64;
  typedef uint32_t words __attribute__((ext_vector_type(2 * DPL)));
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15;
  const int chunks = (p.tokens + 63) / 64, head = block / (chunks * p.share), in_head = block - head * (chunks * p.share);
  const int worker = in_head / chunks, t0 = (in_head - worker * chunks) * 64;
  auto slot_of = [&](int t) {
    if (t < 0 || t >= p.tokens || p.positions[t] < 0) return -2;
    const int s = p.slots[t];
    return s >= 0 && s < p.limit ? s : -2;
  };
  // which of 64 tokens go on the run of the token before, and which of the 16 behind them
  const int mine = slot_of(t0 + lane), last = slot_of(t0 - 1), next = slot_of(lane < 16 ? t0 + 64 + lane : p.tokens);
  int before = __shfl_up(mine, 1, 64), ahead = __shfl_up(next, 1, 64);
  if (lane == 0) before = last;
  if (lane == 0) ahead = __builtin_amdgcn_readlane(mine, 63);
  const bool goes_on = mine >= 0 && (mine & 15) != 0 && mine == before + 1;
  const uint64_t on = __ballot(goes_on), on_next = __ballot(next >= 0 && (next & 15) != 0 && next == ahead + 1);
  const bool leads = mine >= 0 && !goes_on;
  const uint64_t runs = __ballot(leads);
  const int rank = __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(runs >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(runs), 0));
  const int count = __popcll(runs);
  for (int turn = 4 * worker + w; turn < count; turn += 4 * p.share) {
    const int at0 = __builtin_ctzll(__ballot(leads && rank == turn)), first = t0 + at0;
    const int slot = __builtin_amdgcn_readlane(mine, at0);
    const uint64_t rest = at0 == 63 ? on_next : (on >> (at0 + 1)) | (on_next << (63 - at0));
    const int lo = slot & 15, hi = lo + 1 + __builtin_ctzll(~rest);  // a run ends with its 16 slots
    const int64_t at = ((static_cast<int64_t>(slot >> p.shift) * p.kv_heads + head) << p.shift) + (slot & ((1 << p.shift) - 16));
    words *to = reinterpret_cast<words *>(p.vc + at * (D / 2) + 8 * DPL * lane);
    words old = {};
    if (hi - lo < 16) old = *to;
    uint32_t x[16];
#pragma unroll
    for (int o = 0; o < 16; ++o) {
      x[o] = 0;
      if (o >= lo && o < hi) {
        const bf16 *src = p.v + (first + o - lo) * p.v_stride + head * D + DPL * lane;
        if constexpr (DPL == 2) x[o] = *reinterpret_cast<const uint32_t *>(src);
        else x[o] = *reinterpret_cast<const uint16_t *>(src);
      }
    }
    // the largest of each token's group: magnitude bits and whether positive, two tokens to a register
    uint32_t key[8];
#pragma unroll
    for (int o = 0; o < 16; ++o) {
      const uint32_t y = ((x[o] & 0x7fff7fffu) << 1) | ((~x[o] >> 15) & 0x00010001u);
      const uint32_t most = DPL == 2 ? max(y & 0xffffu, y >> 16) : y & 0xffffu;
      key[o >> 1] = o & 1 ? key[o >> 1] | (most << 16) : most;
    }
    auto both = [](uint32_t a, uint32_t b) {
      return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
    };
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      key[i] = over8(key[i], both);
      key[i] = both(key[i], dpp<0x140>(key[i]));  // row_mirror
      key[i] = both(key[i], static_cast<uint32_t>(__shfl_xor(static_cast<int>(key[i]), 16, 64)));
      if constexpr (DPL == 1) key[i] = both(key[i], static_cast<uint32_t>(__shfl_xor(static_cast<int>(key[i]), 32, 64)));
    }
    uint32_t own = key[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) own = (c >> 1) == i ? key[i] : own;
    own = c & 1 ? own >> 16 : own & 0xffffu;
    // as an fp32 number's key
    const float s = kv4_scale(((own >> 1) << 17) | (own & 1)), inv = kv4_inverse(s);
    uint32_t keep[2] = {0, 0};  // nibbles of other tokens
    words out = {};
    each16([&](auto t) {
      constexpr int T = decltype(t)::value, J = 4 * w4_nibble(T & 7), H = T >> 3;
      const float st = row_lane<T>(s), it = row_lane<T>(inv);
      if (!(T >= lo && T < hi)) keep[H] |= 15u << J;
#pragma unroll
      for (int e = 0; e < DPL; ++e) {
        const float y = __uint_as_float(e ? x[T] & 0xffff0000u : x[T] << 16);
        uint32_t code = kv4_code<1>(y, st, it);
        if (!(st == st)) code = 8;
        out[2 * e + H] |= code << J;
      }
    });
#pragma unroll
    for (int e = 0; e < DPL; ++e)
#pragma unroll
      for (int h = 0; h < 2; ++h) out[2 * e + h] = (old[2 * e + h] & keep[h]) | (out[2 * e + h] & ~keep[h]);
    *to = out;
    if ((lane & 16) == 0 && (DPL == 2 || lane < 16) && c >= lo && c < hi) p.vs[(at + c) * NG + (DPL == 2 ? lane >> 5 : 0)] = static_cast<bf16>(s);
  }
}

template <int D>
__global__ __launch_bounds__(256) void kv4_append(Kv4AppendArgs p) {
  const int block = blockIdx.x;
  if (block < p.rows_grid) kv4_rows<D>(p, block);
  else kv4_values<D>(p, block - p.rows_grid);
}

}  // namespace teeny

using namespace teeny;

extern "C" {

teeny_status teeny_kv4_cache_append(const void *q, const void *k, const void *v, const int32_t *positions,
                                    const int32_t *slots, const float *inv_freq, void *q_out, int8_t *k_cache,
                                    int8_t *v_cache, void *k_scale, void *v_scale, int64_t n_tokens, int64_t q_heads,
                                    int64_t kv_heads, int64_t head_dim, int64_t rotary_dim, int64_t num_pages,
                                    int64_t page_size, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                    int32_t interleaved, teeny_stream stream) {
  const char *nm = "kv4_cache_append";
  TEENY_REQUIRE(n_tokens >= 0 && q_heads >= 0 && kv_heads >= 0 && num_pages >= 0 && rotary_dim >= 0,
                TEENY_ERR_SHAPE_MISMATCH, "kv4_cache_append: negative size");
  TEENY_REQUIRE(head_dim == 64 || head_dim == 128, TEENY_ERR_UNSUPPORTED, "kv4_cache_append: head_dim must be 64 or 128");
  TEENY_REQUIRE(rotary_dim % 16 == 0 && rotary_dim <= head_dim, TEENY_ERR_UNSUPPORTED,
                "kv4_cache_append: rotary_dim must be a multiple of 16 up to head_dim");
  const int shift = kv_page_shift(page_size);
  TEENY_REQUIRE(shift > 0, TEENY_ERR_UNSUPPORTED, "kv4_cache_append: page_size must be 16, 32, 64 or 128");
  TEENY_REQUIRE(num_pages <= 0x7fffffff / page_size && n_tokens <= 1 << 24 && q_heads <= 65535 && kv_heads <= 65535,
                TEENY_ERR_SHAPE_MISMATCH, "kv4_cache_append: slots exceed 2^31-1, tokens 2^24 or heads 65535");
  if (num_pages == 0) kv_heads = 0;
  if (n_tokens == 0 || (q_heads == 0 && kv_heads == 0)) return TEENY_OK;
  TEENY_REQUIRE(positions != nullptr && (rotary_dim == 0 || inv_freq != nullptr), TEENY_ERR_NULL_POINTER,
                "kv4_cache_append: positions/inv_freq");
  TEENY_REQUIRE(q_heads == 0 || (q != nullptr && q_out != nullptr), TEENY_ERR_NULL_POINTER, "kv4_cache_append: q/q_out");
  TEENY_REQUIRE(kv_heads == 0 || (k != nullptr && v != nullptr && slots != nullptr && k_cache != nullptr &&
                                  v_cache != nullptr && k_scale != nullptr && v_scale != nullptr),
                TEENY_ERR_NULL_POINTER, "kv4_cache_append: k/v/slots/cache/scale");
  TEENY_REQUIRE((q_heads == 0 || q_stride >= q_heads * head_dim) &&
                    (kv_heads == 0 || (k_stride >= kv_heads * head_dim && v_stride >= kv_heads * head_dim)),
                TEENY_ERR_SHAPE_MISMATCH, "kv4_cache_append: token strides below heads * head_dim");
  // Workgroups of rows take a token, of more than 512 tokens four, which share the angles' work (1 / 4 tokens, 32 and 8 heads of
  // 128: 300 tokens 6.4 / 7.4 us, 900 11.0 / 9.1, 8000 56 / 44).  V's 64 tokens of a head may be 64 runs, in a decode step, or
  // four: workgroups to them by the number of tokens (4 / 8 / 16 of them: 64 tokens of their own 10.4 / 6.5 / 4.5 us, 256
  // 12.3 / 8.4 / 6.7, 80 in runs of five, 16 heads of 64 4.8 / 5.0 / 5.5; 1 / 2 / 4 / 8: 8000 tokens 44.3 / 44.3 / 46 / 51, 500
  // 8 / 16 9.8 / 11.0).
  const int per = n_tokens > 512 ? 4 : 1;
  int share = n_tokens <= 256 ? 16 : n_tokens <= 1024 ? 8 : 2;
  const int64_t rows = cdiv(n_tokens, per), values = cdiv(n_tokens, 64) * kv_heads, most = int64_t{1} << 23;
  while (share > 1 && rows + values * share >= most) share /= 2;  // thousands of heads
  const int64_t all = rows + values * share;
  TEENY_REQUIRE(all < most, TEENY_ERR_SHAPE_MISMATCH, "kv4_cache_append: too many rows for a launch");
  TEENY_REQUIRE(aligned(q, 16) && aligned(q_out, 16) && aligned(k, 16) && aligned(v, 16) && aligned(k_cache, 16) &&
                    aligned(v_cache, 16) && (q_heads == 0 || q_stride % 8 == 0) &&
                    (kv_heads == 0 || (k_stride % 8 == 0 && v_stride % 8 == 0)),
                TEENY_ERR_MISALIGNED, "kv4_cache_append: 16-byte aligned tensors and token strides");
  // each row's numbers are read by the lanes that write them, but rows of another stride lie elsewhere
  TEENY_REQUIRE(q_heads == 0 || q != q_out || q_stride == q_heads * head_dim, TEENY_ERR_INVALID_ARGUMENT,
                "kv4_cache_append: q_out can be q only where q's rows are dense");
  Kv4AppendArgs p{static_cast<const bf16 *>(q), static_cast<const bf16 *>(k), static_cast<const bf16 *>(v), q_stride,
                  k_stride, v_stride, positions, slots, inv_freq, static_cast<bf16 *>(q_out), k_cache, v_cache,
                  static_cast<bf16 *>(k_scale), static_cast<bf16 *>(v_scale), static_cast<int>(n_tokens),
                  static_cast<int>(q_heads), static_cast<int>(kv_heads), static_cast<int>(num_pages << shift), shift,
                  static_cast<int>(rotary_dim / 2), interleaved != 0, 1, 0, 1};
  p.per = per;
  p.share = share;
  p.rows_grid = static_cast<int>(rows);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(all));
  if (head_dim == 64) hipLaunchKernelGGL(kv4_append<64>, grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL(kv4_append<128>, grid, dim3(256), 0, s, p);
  return after_launch(nm, s);
}

}  // extern "C"
