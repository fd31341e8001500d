// Attention over the 4-bit paged K/V cache (kv4_cache.hip), bf16 queries.
//
//   s = softmax_scale sum_G ks[token, G] (q_G . kq_G),  o_G = sum softmax(s) vs[token, G] vq_G
//
// G: groups of 64 numbers of a head.  Ragged batches, grouped heads and the
// dealing out of rows, tokens and splits as in kv_attn.hip; no counterpart in the
// reference (flash_attn2.rs:52-158 reads dense K and V).
//
// A wave takes 64 tokens a time, 16 to each of its four lane groups, as the rows
// of S^T = K Q^T and the k's of O^T += V^T P^T on v_mfma_f32_16x16x32_bf16: lane
// group g's scores are tokens 16 g .. 16 g + 15 of one query, and the
// probabilities are the next product's operand in the registers they were made
// in.  The cache is laid out for this: a lane's 16 bytes are its operands of one
// token's K row, or of two of V's d's over 16 tokens, so codes come straight from
// memory, each byte to one lane: no LDS and no barrier in the loop.
//
// The codes' way to operands, of which there are more than bytes from memory, is
// what it takes beside the reading.  Of up to 16 rows the keys are fp8 operands,
// where a nibble is a number as it stands (w4_fp8), and a query is the sum of two
// fp8 ones, which leaves an error of 2^-17 of its row's largest number; the 8 too
// much is -8 times the sum of q, which the scores start from.  Values, and keys of 17
// to 64 rows, become the bf16 numbers (24 + code) / 16 with two instructions a pair
// (W4Bits), exact; the 24/16 too much is -1.5 times the sum of what they are
// multiplied with, one more product with a constant operand.  Scales are applied in
// fp32: K's to the group's scores, V's to the probability before its rounding to bf16
// (the one rounding on the way, as in kv_attn).  Lane c of a group holds the scale of
// the group's token c, and the multiplication fetches it across the 16 lanes
// (row_newbcast).  For 64 tokens of 128 numbers a wave reads 8.7 KB and issues 360
// vector instructions and 52 products.  One query to each of 64 contexts of 90 to
// 8000 tokens, 32 heads over 8 of 128: 68 us, 4.1 TB/s, for want of waves at the end;
// of 8000 tokens each 122 us, 4.6 TB/s, in the two splits that serve ragged contexts
// (unsplit 107 us, 5.2 TB/s, the rate of a copy).  17 to 64 rows: five queries to each
// of 16 contexts of 3000 tokens, 64 heads over 8 of 128, 39.5 us, 1.4 TB/s: two blocks of
// rows read and unpack the cache each, with 128 products for 64 tokens; vector
// instructions take 59 % of the SIMDs' cycles and products 34 %, with 1.7 waves (of two
// that 242 registers allow) to do one beside the other.
#include "kv4.hpp"
#include "kv_attn.hpp"

namespace teeny {

struct Kv4AttnArgs : KvAttnArgs {
  const bf16 *ks, *vs;
  int sorted;  // parts in order of their length
};

// Part u of a head, one split of one row block, the longest parts first (in eighths of a split), for up to 64 sequences:
// a later, longer part would run on alone when the others are done.  Lane b counts its sequence's parts that are longer
// than tau eighths; they are the first ones of the order: whole splits, then the rest of the context.
template <int RB>
__device__ __forceinline__ bool kv4_parts_sorted(const KvAttnArgs &p, int u, KvRows &r, int &split) {
  const int lane = threadIdx.x & 63, b = min(lane, p.batch - 1);
  auto start = [&](int i) { return min(max(p.starts ? p.starts[i] : i, 0), p.tokens); };
  const int first = start(b), len = lane < p.batch ? max(start(b + 1) - first, 0) : 0;
  const int nb = (len * p.group + RB - 1) / RB, ctx = min(max(p.ctx[b], 0), p.width << p.shift);
  const int full = min(ctx / p.chunk, p.splits), rest = full < p.splits ? ctx - full * p.chunk : 0, eighth = p.chunk / 8;
  auto count = [&](int tau) -> uint32_t {
    if (tau == 0) return nb * max(full + (rest > 0), 1);
    return nb * ((tau <= 8 ? full : 0) + (rest > (tau - 1) * eighth && tau <= 8));
  };
  auto total = [&](uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(wave_scan(v)), 63)); };
  if (total(count(0)) <= static_cast<uint32_t>(u)) return false;
  int lo = 0, hi = 9;  // total(count(lo)) > u >= total(count(hi)) = 0
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (total(count(mid)) > static_cast<uint32_t>(u)) lo = mid;
    else hi = mid;
  }
  const uint32_t above = count(hi), here = count(lo) - above, upto = wave_scan(here);
  const uint32_t at = u - total(above);
  const int owner = __builtin_ctzll(__ballot(upto > at));
  auto from = [&](int v) { return __builtin_amdgcn_readlane(v, owner); };
  const int blocks = from(nb), part = from(above) + at - (from(upto) - from(here));
  r.b = owner;
  r.first = from(first);
  r.len = from(len);
  r.rows = r.len * p.group;
  r.ctx = from(ctx);
  split = part / blocks;
  r.row0 = (part - split * blocks) * RB;
  return true;
}

// Codes as fp8 (e4m3): the bytes 0 .. 15 are the numbers 0 .. 15 times 2^-9, since denormal numbers and the first
// normal ones lie equally far apart.  So a nibble is its operand as it is, in the order of fp8_order.
__device__ __forceinline__ int64_t w4_fp8(uint32_t word) {
  const uint32_t even = word & 0x0f0f0f0fu, odd = (word >> 4) & 0x0f0f0f0fu;
  return static_cast<int64_t>(static_cast<uint64_t>(odd) << 32 | even);
}
__device__ constexpr int fp8_order(int byte) { return (byte & 1) * 4 + (byte >> 1); }

// Eight numbers as the sum of two fp8 ones each, bytes in fp8_order.  Of numbers up to 256 the first takes four bits of
// significand, the second what is left, down to 2^-9.
__device__ __forceinline__ void fp8_parts(const float (&v)[8], int64_t &first, int64_t &second) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  uint32_t part[2][2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = v[fp8_order(4 * h + i)];
    int a = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    a = __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], a, true);
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(a, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(a, true);
    int b = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] - lo[0], x[1] - lo[1], 0, false);
    b = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] - hi[0], x[3] - hi[1], b, true);
    part[0][h] = a;
    part[1][h] = b;
  }
  first = static_cast<int64_t>(static_cast<uint64_t>(part[0][1]) << 32 | part[0][0]);
  second = static_cast<int64_t>(static_cast<uint64_t>(part[1][1]) << 32 | part[1][0]);
}
__device__ __forceinline__ f32x4 mfma16_fp8(int64_t a, int64_t b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_fp8_fp8(a, b, c, 0, 0, 0);
}

// V scales from kVast on could overflow the sums of p v, where p is up to 2^8 and there may be 2^30 tokens.  Once a wave
// meets one that a row of its block sees, the exponents' reference lies kRaise above the scores' maximum: p, l and the sums
// are all by 2^-kRaise smaller, and every join of parts goes by that reference.  (Beside such a scale, values below 2^-70
// fall below bf16's and fp32's smallest numbers.)
constexpr float kVast = 0x1p80f, kRaise = 48.0f;

// The least that scores are multiplied with, so that a masked -inf gives p = 0 under a zero scale too.  (It is the smallest
// number: times the largest score it is 2^-21, where FLT_MIN gave 4.)
constexpr float kLeast = 0x1p-149f;

// Whether one of a token's V scales is kVast or more, or no number: by its bits.
template <int NG, typename S>
__device__ __forceinline__ bool kv4_vast(S scales) {
  constexpr uint32_t vast = 0x6780;  // 2^80
  if constexpr (NG == 1) {
    return (__builtin_bit_cast(uint16_t, scales) & 0x7fffu) >= vast;
  } else {
    const uint32_t both = __builtin_bit_cast(uint32_t, scales);
    return (both & 0x7fffffffu) >= vast << 16 || (both & 0x7fffu) >= vast;
  }
}

// NQ: 16-row column blocks; the four waves share out the tokens, 64 a time.
template <int D, int NQ>
__global__ __launch_bounds__(256, 2) void kv4_attn(Kv4AttnArgs p) {
  constexpr int WK = 4, WROWS = 16 * NQ, RB = WROWS;
  constexpr int NC = D / 32, ND = D / 16, NG = D / 64, NV = D / 32;  // k-steps of the scores, d blocks, groups, V vectors
  constexpr int LD = D + 4;
  constexpr bool FP8 = NQ == 1;  // keys as fp8 operands
  typedef uint32_t kvec __attribute__((ext_vector_type(2 * NG)));
  typedef __bf16 svec __attribute__((ext_vector_type(NG)));
  __shared__ __attribute__((aligned(16))) float red[WK * WROWS * LD];
  __shared__ float ml[2][WK][WROWS];
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  // the blocks that the caller's lengths stand for come first, then those that there may be beyond, mostly none
  const int per_block = p.splits * p.kv_heads, first = p.walk * per_block;
  const bool beyond = static_cast<int>(blockIdx.x) >= first;
  const int id = beyond ? blockIdx.x - first : xcd_remap(blockIdx.x, first), of = beyond ? p.blocks - p.walk : p.walk;
  const int head = id / (p.splits * of), in_head = id - head * (p.splits * of);
  int split = in_head / of;
  KvRows r;
  if (p.sorted) {
    if (!kv4_parts_sorted<RB>(p, in_head + (beyond ? p.walk * p.splits : 0), r, split)) return;
  } else if (!kv_rows<RB>(p, in_head - split * of + (beyond ? p.walk : 0), r)) {
    return;
  }
  // row i of the sequence: query i / group, head i % group of the K/V head's; it sees seen(i) tokens
  auto seen = [&](int i) { return p.causal ? min(max(r.ctx - r.len + 1 + i / p.group, 0), r.ctx) : r.ctx; };
  const int k_end = seen(min(r.row0 + RB, r.rows) - 1);
  // the last split takes what lies past the longest context that the caller expected
  const int kb = split * p.chunk, ke = split == p.splits - 1 ? k_end : min(k_end, kb + p.chunk);
  if (split > 0 && kb >= k_end) return;

  const int32_t *row = p.table + static_cast<int64_t>(r.b) * p.width;
  const int page_mask = (1 << p.shift) - 1;
  struct Pages {
    int k, v;  // pages of the lane's K rows and V columns, -1: none
  };
  auto page_at = [&](int t) {
    const int pg = row[min(t, k_end - 1) >> p.shift];
    return t < k_end && pg >= 0 && pg < p.pages ? pg : -1;
  };
  auto load_pages = [&](int t0) { return Pages{page_at(t0 + 16 * (c >> 2)), page_at(t0 + 16 * g)}; };
  // a page's tokens of this head, as tokens of the whole cache
  auto token_at = [&](int page, int t) {
    return ((static_cast<int64_t>(max(page, 0)) * p.kv_heads + head) << p.shift) + (t & page_mask);
  };
  kvec kr[4];
  u32x4 vr[NV];
  svec ks, vs;
  bool none = false;
  auto load_k = [&](int t0, Pages pg) {
    const int8_t *src = p.kc + (token_at(pg.k, t0 + 16 * (c >> 2)) + (c & 3)) * (D / 2) + (D / 8) * g;
#pragma unroll
    for (int i = 0; i < 4; ++i) kr[i] = *reinterpret_cast<const kvec *>(src + 4 * i * (D / 2));
  };
  auto load_v = [&](int t0, Pages pg) {
    const int64_t at = token_at(pg.v, t0 + 16 * g);
    const int8_t *src = p.vc + at * (D / 2) + 16 * c;
#pragma unroll
    for (int a = 0; a < NV; ++a) vr[a] = *reinterpret_cast<const u32x4 *>(src + 256 * a);
    ks = *reinterpret_cast<const svec *>(p.ks + (at + c) * NG);
    vs = *reinterpret_cast<const svec *>(p.vs + (at + c) * NG);
    none = pg.v < 0;
  };
  constexpr int STEP = 64 * WK;
  int t0 = kb + 64 * w;
  Pages pg;
  if (t0 < ke) {
    pg = load_pages(t0);
    load_k(t0, pg);
    load_v(t0, pg);
    pg = load_pages(t0 + STEP);
  }

  const uint32_t qsign = p.scale_log2 < 0.0f ? 0x80008000u : 0u;  // a negative scale's sign goes to Q
  const u32x4 off_bits = u32x4{0xBFC0BFC0u, 0xBFC0BFC0u, 0xBFC0BFC0u, 0xBFC0BFC0u};  // -1.5
  const bf16x8 off = __builtin_bit_cast(bf16x8, off_bits);
  const W4Bits w4;
  bf16x8 qf[FP8 ? 1 : NQ][FP8 ? 1 : NC];
  int64_t q8[FP8 ? NC : 1][2];
  f32x4 q_off[FP8 ? NG : 1];  // -8 sum of q over the group (times 2^-9), in every row
  float col[NQ];              // what the column's scores are to be multiplied with, softmax_scale among it
  int vis[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int i = min(r.row0 + 16 * n + c, r.rows - 1), t = i / p.group;
    vis[n] = p.causal ? min(max(r.ctx - r.len + 1 + t, 0), r.ctx) : r.ctx;
    const int h = head * p.group + i - t * p.group;
    const bf16 *at = p.q + (r.first + t) * p.q_stride + h * D;
    u32x4 raw[NC];
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      raw[j] = *reinterpret_cast<const u32x4 *>(at + (j >> 1) * 64 + g * 16 + (j & 1) * 8);
      raw[j] ^= qsign;
    }
    float scale = 16.0f * fabsf(p.scale_log2);  // 16: of W4Bits
    if constexpr (FP8) {
      // the row's largest number to 128 .. 256 by a power of two; an infinity or NaN makes all of it NaN
      uint32_t most = 0;
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) most = max(most, max(raw[j][e] & 0x7fffu, raw[j][e] >> 16 & 0x7fffu));
      most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 16, 64)));
      most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 32, 64)));
      const int exponent = max(static_cast<int>(most >> 7), 8);  // biased; below: numbers that lose bits beside 2^-119
      const float up = most >= 0x7f80u ? __uint_as_float(0x7fc00000u) : __uint_as_float(static_cast<uint32_t>(127 + 127 + 7 - exponent) << 23);
      scale = __builtin_ldexpf(fabsf(p.scale_log2), exponent - 134 + 9);  // over `up` and 2^-9
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[2 * e] = __uint_as_float(raw[j][e] << 16) * up;
          v[2 * e + 1] = __uint_as_float(raw[j][e] & 0xffff0000u) * up;
        }
        fp8_parts(v, q8[j][0], q8[j][1]);
      }
#pragma unroll
      for (int G = 0; G < NG; ++G) {
        q_off[G] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        const int64_t minus8 = static_cast<int64_t>(0x8888888888888888ull);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int b = 0; b < 2; ++b) q_off[G] = mfma16_fp8(minus8, q8[2 * G + j][b], q_off[G]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < NC; ++j) qf[n][j] = __builtin_bit_cast(bf16x8, raw[j]);
    }
    col[n] = scale;
  }
  // Beside a query of up to 256 K scales near the largest number could overflow the scores, before `col`: they are taken
  // 2^-12 of.  (Where `col` is so large that it could not make up for it, such scores overflow anyway.)
  const float down = FP8 && !__any(col[0] >= 0x1p100f) ? 0x1p-12f : 1.0f;
  col[0] *= 1.0f / down;
#pragma unroll
  for (int n = 0; n < NQ; ++n) col[n] = fmaxf(col[n], kLeast);
  const int all_see = seen(r.row0);  // all rows see the tokens below it

  f32x4 acc[NQ][ND], p_off[FP8 ? NG : 1];  // p_off: -1.5 sum of the weighted probabilities, in every row
  float m_run[NQ], l_run[NQ], raise = 0.0f;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    m_run[n] = -INFINITY;
    l_run[n] = 0.0f;
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[n][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (FP8)
#pragma unroll
      for (int G = 0; G < NG; ++G) p_off[G] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
#pragma unroll 1
  for (; t0 < ke; t0 += STEP) {
    if (__any(kv4_vast<NG>(vs)) && __any(kv4_vast<NG>(vs) && !none && t0 + 16 * g + c < k_end)) raise = kRaise;
    float ksc[NG], vsc[NG];  // of the lane group's token c
#pragma unroll
    for (int G = 0; G < NG; ++G) {
      const float k = static_cast<float>(ks[G]);
      ksc[G] = FP8 ? __builtin_fmaf(k, down, k * 0.0f) : __builtin_fmaf(k, 0.0f, k);  // an infinity counts as NaN
      vsc[G] = static_cast<float>(vs[G]);
    }
    f32x4 s[NQ][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int G = 0; G < NG; ++G) {
        f32x4 xs[NQ];
        if constexpr (FP8) {
          xs[0] = q_off[G % (FP8 ? NG : 1)];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int64_t a = w4_fp8(kr[i][2 * G + j]);
#pragma unroll
            for (int b = 0; b < 2; ++b) xs[0] = mfma16_fp8(a, q8[(2 * G + j) % (FP8 ? NC : 1)][b], xs[0]);
          }
        } else {
          // (no registers to spare for the offsets: the products that give them are made again)
          const bf16x8 a0 = w4.values(kr[i][2 * G]), a1 = w4.values(kr[i][2 * G + 1]);
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            const bf16x8 *q = qf[n % (FP8 ? 1 : NQ)];
            const int j = (2 * G) % (FP8 ? 1 : NC), k = (2 * G + 1) % (FP8 ? 1 : NC);
            xs[n] = mfma16(a1, q[k], mfma16(a0, q[j], f32x4{0.0f, 0.0f, 0.0f, 0.0f}));
            xs[n] = mfma16(off, q[k], mfma16(off, q[j], xs[n]));
          }
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          const f32x4 x = xs[n];
          each16([&](auto t) {
            constexpr int T = decltype(t)::value;
            if (T >> 2 == i) {
              const float sc = row_lane<T>(ksc[G]);
              s[n][i][T & 3] = G == 0 ? sc * x[T & 3] : __builtin_fmaf(sc, x[T & 3], s[n][i][T & 3]);
            }
          });
        }
      }
      // scaled here and now, or the scaling sinks below the branch, away from the lanes it takes the scales from
#pragma unroll
      for (int n = 0; n < NQ; ++n) asm volatile("" : "+v"(s[n][i]));
      __builtin_amdgcn_sched_barrier(0);
    }
    const bool more = t0 + STEP < ke;
    const bool hidden = none;
    if (more) load_k(t0 + STEP, pg);
    const bool masks = t0 + 64 > all_see || __any(hidden);
    const int at = t0 + 16 * g;  // the lane's first token
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      if (masks) {  // also the scores of scales that may be anything
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (hidden || at + i >= vis[n]) s[n][i >> 2][i & 3] = -INFINITY;
      }
      float mx = s[n][0][0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = __builtin_elementwise_maximum(mx, s[n][i >> 2][i & 3]);
      mx = over_groups(__builtin_fmaf(mx, col[n], raise), [](float a, float b) { return __builtin_elementwise_maximum(a, b); });
      if (__any(mx > m_run[n] + 8.0f)) {  // rescaled rarely: p <= 2^8
        const float m_new = fmaxf(m_run[n], mx);
        const float alpha = __builtin_amdgcn_exp2f(m_run[n] - (m_new == -INFINITY ? 0.0f : m_new));
        l_run[n] *= alpha;
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[n][d] *= alpha;
        if constexpr (FP8)
#pragma unroll
          for (int G = 0; G < NG; ++G) p_off[G] *= alpha;
        m_run[n] = m_new;
      }
      const float neg_m = m_run[n] == -INFINITY ? 0.0f : -m_run[n];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][i >> 2][i & 3], col[n], neg_m));
        l_run[n] += e;
        s[n][i >> 2][i & 3] = e;
      }
    }
#pragma unroll
    for (int G = 0; G < NG; ++G) {
      bf16x8 pb[NQ][2];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        float v[16];
        each16([&](auto t) {
          constexpr int T = decltype(t)::value;
          v[T] = s[n][T >> 2][T & 3] * row_lane<T>(vsc[G]);
        });
        if (masks) {  // a hidden token's V scale may be anything
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (hidden || at + i >= vis[n]) v[i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const bf16x2 pr = cvt_pk_bf16(v[i], v[i + 1]);
          pb[n][i >> 3][i & 7] = pr[0];
          pb[n][i >> 3][(i & 7) + 1] = pr[1];
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (FP8) p_off[G % (FP8 ? NG : 1)] = mfma16(off, pb[0][h], p_off[G % (FP8 ? NG : 1)]);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const bf16x8 a = w4.values(vr[2 * G + (d >> 1)][2 * (d & 1) + h]);
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            acc[n][4 * G + d] = mfma16(a, pb[n][h], acc[n][4 * G + d]);
            if constexpr (!FP8) acc[n][4 * G + d] = mfma16(off, pb[n][h], acc[n][4 * G + d]);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (more) {
      load_v(t0 + STEP, pg);
      pg = load_pages(t0 + 2 * STEP);
    }
  }
#pragma unroll
  for (int n = 0; n < NQ; ++n) l_run[n] = over_groups(l_run[n], [](float a, float b) { return a + b; });

  // the waves' parts: a common max, then the sum of their outputs in wave order
  const bool whole = p.part == nullptr || k_end <= p.chunk;  // no other split has a part of these rows
  const int64_t unit = static_cast<int64_t>(head) * p.blocks + r.number<RB>(p);
  const int64_t slot = (unit * p.splits + split) * RB;  // part rows of this (unit, split)
  if (g == 0) {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      ml[0][w][16 * n + c] = m_run[n];
      ml[1][w][16 * n + c] = l_run[n];
    }
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int at = 16 * n + c;
    float m = ml[0][0][at], l = 0.0f;
#pragma unroll
    for (int i = 1; i < WK; ++i) m = fmaxf(m, ml[0][i][at]);
    const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int i = 0; i < WK; ++i) l += ml[1][i][at] * __builtin_amdgcn_exp2f(ml[0][i][at] - ref);
    const float mul = 16.0f * __builtin_amdgcn_exp2f(m_run[n] - ref) * (whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f);
    // blocks 2 a and 2 a + 1 hold the even and odd d's of 32 a ..: the lane's are eight consecutive ones
#pragma unroll
    for (int a = 0; a < NV; ++a) {
      f32x4 even = acc[n][2 * a], odd = acc[n][2 * a + 1];
      if constexpr (FP8) even += p_off[(a >> 1) % (FP8 ? NG : 1)], odd += p_off[(a >> 1) % (FP8 ? NG : 1)];
      even *= mul, odd *= mul;
      float *to = red + (w * WROWS + at) * LD + 32 * a + 8 * g;
      *reinterpret_cast<f32x4 *>(to) = f32x4{even[0], odd[0], even[1], odd[1]};
      *reinterpret_cast<f32x4 *>(to + 4) = f32x4{even[2], odd[2], even[3], odd[3]};
    }
    if (w == 0 && g == 0 && r.row0 + at < r.rows) {
      if (!whole) {
        p.part[p.ml_off + (slot + at) * 2] = m;
        p.part[p.ml_off + (slot + at) * 2 + 1] = l;
      } else if (p.l != nullptr) {
        const int t = (r.row0 + at) / p.group;
        p.l[static_cast<int64_t>(r.first + t) * p.heads + head * p.group + r.row0 + at - t * p.group] = (m + log2f(l)) * 0.6931471805599453f;
      }
    }
  }
  __syncthreads();
  const int rows = min(WROWS, r.rows - r.row0);
  for (int i = threadIdx.x; i < rows * (D / 4); i += 256) {
    const int at = i / (D / 4), d = 4 * (i % (D / 4));
    f32x4 o = *reinterpret_cast<const f32x4 *>(red + at * LD + d);
#pragma unroll
    for (int k = 1; k < WK; ++k) o += *reinterpret_cast<const f32x4 *>(red + (k * WROWS + at) * LD + d);
    if (whole) {
      const int t = (r.row0 + at) / p.group, h = head * p.group + (r.row0 + at) - t * p.group;
      bf16x4 o4;
#pragma unroll
      for (int v = 0; v < 4; ++v) o4[v] = static_cast<bf16>(o[v]);
      *reinterpret_cast<bf16x4 *>(p.o + (static_cast<int64_t>(r.first + t) * p.heads + h) * D + d) = o4;
    } else {
      *reinterpret_cast<f32x4 *>(p.part + (slot + at) * D + d) = o;
    }
  }
}

// Eight codes of a word as code / 16 times eight scales.
template <typename S>
__device__ __forceinline__ bf16x8 kv4_values8(uint32_t word, S scale) {
  const uint32_t even = word ^ 0x88888888u;  // two's complement nibbles
  uint32_t odd = even >> 4;
  asm("" : "+v"(odd));  // a byte of it is an operand as it is, of word >> 4 a shift more
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int n = w4_nibble(j);
    v[j] = __builtin_amdgcn_cvt_off_f32_i4(static_cast<int>((n & 1 ? odd : even) >> (8 * (n >> 1)) & 0xffu));
  }
  scale(v);
  bf16x8 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bf16x2 pr = cvt_pk_bf16(v[2 * j], v[2 * j + 1]);
    r[2 * j] = pr[0];
    r[2 * j + 1] = pr[1];
  }
  return r;
}

// Many query rows (prompts in pieces): bound by the products and the work beside
// them.  As in kv_attn_tile a workgroup of eight waves, 32 rows each, turns a tile of
// 64 tokens once into the bf16 operands of v_mfma_f32_32x32x16_bf16, in LDS in the
// order in which lanes take them up; here code times scale, a bf16 number already
// where the scale has five bits (other scales: rounded), so that the products need
// no scale of their own.  The next tile is turned while one is multiplied, the codes
// of the tile after that are in flight; one barrier a tile.  Bound by the vector instructions, 290 a wave and tile, 32 of
// them exponentials (62 % of the SIMDs' cycles), beside 32 products of 32 cycles (44 %): 4 requests of 700 queries and
// 1100 to 4100 tokens, 32 heads of 128 over 8: 122 to 132 us, 705 to 764 TFLOP/s;
// 1900 queries of 6400: 203 to 210 us, 806 to 836.  (Four waves and 128 rows, two workgroups on a CU: every row pays
// for turning twice as often, 174 us to 150.  Two groups of waves half a tile apart: 175
// to 150.  Turning and exponentials between the products: 134 to 140.)
template <int D>
__global__ __launch_bounds__(512, 2) void kv4_attn_tile(Kv4AttnArgs p) {
  constexpr int RB = 256, NS = D / 16, ND = D / 32, NG = D / 64, EPW = D / 32, KW = D / 64, FR = 2 * NS + 4 * ND;
  typedef uint32_t kvec __attribute__((ext_vector_type(KW)));
  __shared__ __attribute__((aligned(16))) u32x4 frag[2][FR * 64];  // K [block][step], then V [d block][block][half]
  // of the tokens turned the first whose V scale is not finite (it is turned to zeros), for each group, and the first whose is
  // kVast or more: a row sees it or later ones at most
  __shared__ int nan_from[NG], vast_from;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 31, g = lane >> 5;
  const int id = xcd_remap(blockIdx.x, gridDim.x);
  const int head = id / (p.splits * p.blocks), in_head = id - head * (p.splits * p.blocks);
  const int split = in_head / p.blocks, u = in_head - split * p.blocks;
  KvRows r;
  if (!kv_rows_sorted<RB>(p, u, r)) return;
  auto seen = [&](int i) { return p.causal ? min(max(r.ctx - r.len + 1 + i / p.group, 0), r.ctx) : r.ctx; };
  const int k_end = seen(min(r.row0 + RB, r.rows) - 1);
  const int kb = split * p.chunk, ke = split == p.splits - 1 ? k_end : min(k_end, kb + p.chunk);
  if (split > 0 && kb >= k_end) return;
  const int base = r.row0 + 32 * w;  // the wave's rows; past r.rows it only helps to turn the tiles

  const float sc = fmaxf(16.0f * fabsf(p.scale_log2), kLeast);  // 16: of kv4_values8
  const uint32_t qsign = p.scale_log2 < 0.0f ? 0x80008000u : 0u;  // a negative scale's sign goes to Q
  const int my = min(base + c, r.rows - 1), qt = my / p.group, qh = head * p.group + my - qt * p.group;
  const int64_t out_row = static_cast<int64_t>(r.first + qt) * p.heads + qh;
  const int vis = seen(my), all_see = seen(min(base, r.rows - 1));
  const int w_end = base < r.rows ? min(ke, seen(min(base + 32, r.rows) - 1)) : 0;
  bf16x8 qf[NS];  // step i: numbers of the K word that a lane of wave 2 x + i / EPW turns into it
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const int e = i % EPW, d = 64 * (e >> 1) + 16 * (2 * (i / EPW) + g) + 8 * (e & 1);
    u32x4 raw = *reinterpret_cast<const u32x4 *>(p.q + (r.first + qt) * p.q_stride + qh * D + d);
    raw ^= qsign;
    // an infinity is NaN, or a row whose scores are all -inf would count as one that sees nothing
#pragma unroll
    for (int j = 0; j < 4; ++j)
      raw[j] |= ((raw[j] & 0x7f80u) == 0x7f80u ? 0x40u : 0u) | ((raw[j] & 0x7f800000u) == 0x7f800000u ? 0x400000u : 0u);
    qf[i] = __builtin_bit_cast(bf16x8, raw);
  }
  f32x16 acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) acc[d] = zero16();
  float m_run = -INFINITY, l_run = 0.0f;

  // The wave's share of a tile: of the K rows of block w / 2 % 2, of their chunks 2 (w % 2) and 2 (w % 2) + 1, the words of
  // group w / 4 (D = 64: word w / 4), and of V block w % 2 of d block w / 2 (D = 64: four waves do).  The four pages of a
  // tile are one load for the wave, from which each lane takes those of its K row and its V tokens.
  const int32_t *row = p.table + static_cast<int64_t>(r.b) * p.width;
  const int page_mask = (1 << p.shift) - 1, wb = (w >> 1) & 1, wk = w >> 2, vd = D == 128 ? w >> 1 : (w >> 1) & 1, vb = w & 1;
  const int k_block = 2 * wb + ((c >> 2) & 1), v_block = 2 * vb + g;  // of 16 tokens, of the tile's four
  const int k_token = 16 * k_block + 4 * (c >> 3) + (c & 3), v_token = 16 * v_block + (lane & 15);
  const int8_t *k_from = p.kc + (D / 8) * (2 * (w & 1) + g) + 4 * KW * wk, *v_from = p.vc + 8 * (32 * vd + c);
  const bf16 *ks_from = p.ks + (D == 128 ? wk : 0), *vs_from = p.vs + (vd >> 1);
  // lane l: the page of tokens 16 (l % 4) .. of a tile
  auto load_pages = [&](int t0) { return row[min(t0 + 16 * (lane & 3), k_end - 1) >> p.shift]; };
  kvec kr;
  u32x2 vr;
  bf16 ks, vs;
  bool there_v;
  uint32_t here_next;  // bit j: the tile's tokens 16 j .. have a page (the first of them is below ke)
  auto load_codes = [&](int t0, int pg) {
    const int of = t0 + 16 * (lane & 3) < ke && static_cast<uint32_t>(pg) < static_cast<uint32_t>(p.pages) ? pg : -1;
    here_next = static_cast<uint32_t>(__ballot(of >= 0)) & 15;
    const int k_page = __builtin_amdgcn_ds_bpermute(4 * k_block, of), v_page = __builtin_amdgcn_ds_bpermute(4 * v_block, of);
    auto token = [&](int page, int t) __attribute__((always_inline)) {  // of the cache; page 0 where there is none
      return ((static_cast<uint64_t>(static_cast<uint32_t>(max(page, 0))) * static_cast<uint32_t>(p.kv_heads) + head) << p.shift) + (t & page_mask);
    };
    const uint64_t k_at = token(k_page, t0 + k_token), v_at = token(v_page, t0 + v_token);
    kr = *reinterpret_cast<const kvec *>(k_from + k_at * (D / 2));
    ks = ks_from[k_at * NG];
    if (D == 128 || w < 4) {
      vr = *reinterpret_cast<const u32x2 *>(v_from + (v_at & ~15ull) * (D / 2));
      vs = vs_from[v_at * NG];
      there_v = v_page >= 0 && t0 + v_token < ke;
    }
  };
  auto turn = [&](int buf, int t0) {
    u32x4 *to = frag[buf];
    const float k = static_cast<float>(ks), k_scale = __builtin_fmaf(k, 0.0f, k);  // an infinity counts as NaN
#pragma unroll
    for (int e = 0; e < KW; ++e)
      to[(wb * NS + EPW * (w & 1) + KW * wk + e) * 64 + lane] =
          __builtin_bit_cast(u32x4, kv4_values8(kr[e], [&](float (&v)[8]) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] *= k_scale;
          }));
    if (D == 64 && w >= 4) return;
    float s = static_cast<float>(vs);
    const bool finite = fabsf(s) < INFINITY;
    // lanes 0 .. 15: tokens 0 .. 15 of the block, 32 .. 47: the others
    const uint64_t odd = __ballot(there_v && !(fabsf(s) < kVast)), fit = __ballot(finite);
    s = there_v && finite ? s : 0.0f;
    const int at = 2 * NS + (vd * 2 + vb) * 2;
    to[at * 64 + lane] = __builtin_bit_cast(u32x4, kv4_values8(vr[0], [&](float (&v)[8]) {
                                              each16([&](auto t) {
                                                if constexpr (t < 8) v[t] *= row_lane<t>(s);
                                              });
                                            }));
    to[(at + 1) * 64 + lane] = __builtin_bit_cast(u32x4, kv4_values8(vr[1], [&](float (&v)[8]) {
                                                    each16([&](auto t) {
                                                      if constexpr (t >= 8) v[t - 8] *= row_lane<t>(s);
                                                    });
                                                  }));
    if (odd != 0) {
      auto note = [&](int *from, uint64_t m) {
        if (m != 0) atomicMin(from, t0 + 32 * vb + __builtin_ctz(static_cast<uint32_t>((m & 0xffffu) | (m >> 32 & 0xffffu) << 16)));
      };
      if ((vd & 1) == 0 && lane == 0) note(&nan_from[vd >> 1], odd & ~fit), note(&vast_from, odd & fit);
    }
  };

  int pg = 0, buf = 0;
  uint32_t here = 0;
  if (threadIdx.x == 0) vast_from = nan_from[0] = nan_from[NG - 1] = 0x7fffffff;
  if (kb < ke) pg = load_pages(kb);
  __syncthreads();
  if (kb < ke) {
    load_codes(kb, pg);
    pg = load_pages(kb + 64);
    turn(0, kb);
    here = here_next;
    if (kb + 64 < ke) {
      load_codes(kb + 64, pg);
      pg = load_pages(kb + 128);
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int t0 = kb; t0 < ke; t0 += 64) {
    const u32x4 *now = frag[buf];
    const uint32_t here_now = here;
    // (the next tile's turning, which may be under way, does not change which side of this tile's end it lies on)
    const int vast_at = vast_from;
    if (t0 + 64 < ke) {
      turn(buf ^ 1, t0 + 64);
      here = here_next;
      if (t0 + 128 < ke) {
        load_codes(t0 + 128, pg);
        pg = load_pages(t0 + 192);
      }
    }
    if (t0 < w_end) {
      // operands are read LA products ahead, V's first ones before the exponentials; the order is kept as written
      constexpr int LA = 4, WIN = LA + 1;
      u32x4 win[WIN];
      auto read = [&](int i) __attribute__((always_inline)) {
        const int j = i - 2 * NS;  // scores: both blocks in turn; outputs: the d blocks in turn
        const int at = i < 2 * NS ? (i & 1) * NS + (i >> 1) : 2 * NS + (j % ND) * 4 + j / ND;
        win[i % WIN] = now[at * 64 + lane];
      };
#pragma unroll
      for (int i = 0; i < LA; ++i) read(i);
      f32x16 s[2] = {zero16(), zero16()};
#pragma unroll
      for (int i = 0; i < 2 * NS; ++i) {
        read(i + LA);
        s[i & 1] = mfma32x32x16(__builtin_bit_cast(bf16x8, win[i % WIN]), qf[i >> 1], s[i & 1]);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (t0 + 64 > all_see || here_now != 15) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int v = 0; v < 16; ++v)
            if (((here_now >> (2 * b + g)) & 1) == 0 || t0 + 32 * b + 16 * g + v >= vis) s[b][v] = -INFINITY;
      }
      float mx = s[0][0];
#pragma unroll
      for (int v = 1; v < 32; ++v) mx = __builtin_elementwise_maximum(mx, s[v >> 4][v & 15]);
      const float raise = vast_at < min(t0 + 64, w_end) ? kRaise : 0.0f;  // once above 0 it stays
      mx = __builtin_fmaf(mx, sc, raise);
      const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
      mx = __builtin_elementwise_maximum(__uint_as_float(both[0]), __uint_as_float(both[1]));
      if (__any(mx > m_run + 8.0f)) {  // rescaled rarely: p <= 2^8
        const float m_new = fmaxf(m_run, mx);
        const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.0f : m_new));
        l_run *= alpha;
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d] *= alpha;
        m_run = m_new;
      }
      const float neg_m = m_run == -INFINITY ? 0.0f : -m_run;
      bf16x8 pb[2][2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          s[b][v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][v], sc, neg_m));
          l_run += s[b][v];
        }
#pragma unroll
        for (int v = 0; v < 16; v += 2) {
          const bf16x2 pr = cvt_pk_bf16(s[b][v], s[b][v + 1]);
          pb[b][v >> 3][v & 7] = pr[0];
          pb[b][v >> 3][(v & 7) + 1] = pr[1];
        }
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < 4 * ND; ++j) {
        const int i = 2 * NS + j, d = j % ND, bh = j / ND;
        if (j + LA < 4 * ND) read(i + LA);
        acc[d] = mfma32x32x16(__builtin_bit_cast(bf16x8, win[i % WIN]), pb[bh >> 1][bh & 1], acc[d]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    buf ^= 1;
    __syncthreads();
  }
  l_run += __shfl_xor(l_run, 32, 64);
  if (base + c >= r.rows) return;
  // a row that sees a token whose V is NaN: its outputs of that group are, whatever the token's weight
#pragma unroll
  for (int G = 0; G < NG; ++G)
    if (nan_from[G] < vis) {
      acc[2 * G] *= __uint_as_float(0x7fc00000u);
      acc[2 * G + 1] *= __uint_as_float(0x7fc00000u);
    }
  const bool whole = p.part == nullptr || k_end <= p.chunk;  // no other split has a part of these rows
  const int64_t unit = static_cast<int64_t>(head) * p.blocks + r.number<RB>(p);
  const int64_t slot = (unit * p.splits + split) * RB + 32 * w + c;
  const float mul = 16.0f * (whole ? (l_run == 0.0f ? 0.0f : 1.0f / l_run) : 1.0f);
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int at = 32 * d + 8 * a + 4 * g;
      f32x4 o = f32x4{acc[d][4 * a], acc[d][4 * a + 1], acc[d][4 * a + 2], acc[d][4 * a + 3]} * mul;
      if (whole) {
        bf16x4 o4;
#pragma unroll
        for (int v = 0; v < 4; ++v) o4[v] = static_cast<bf16>(o[v]);
        *reinterpret_cast<bf16x4 *>(p.o + out_row * D + at) = o4;
      } else {
        *reinterpret_cast<f32x4 *>(p.part + slot * D + at) = o;
      }
    }
  if (g == 0 && !whole) {
    p.part[p.ml_off + slot * 2] = m_run;
    p.part[p.ml_off + slot * 2 + 1] = l_run;
  } else if (g == 0 && p.l != nullptr) {
    p.l[out_row] = (m_run + log2f(l_run)) * 0.6931471805599453f;
  }
}

// ── which form, and how many splits ─────────────────────────────────────────
// Few rows take kv4_attn, more than 64 a sequence the shared tiles.  kv4_attn's splits give a workgroup one round of 256
// tokens where they leave CUs free, two where the device is busier, from three rounds on.  Several sequences, which may
// differ in length, take so many that there are four workgroups to a CU if all are as long as the longest, of 1024 tokens
// or more each, and never more than 8192 tokens to one (of many sequences one may be by far the longest); up to 64 of them
// are dealt out longest first.  us by splits, one query, 8 K/V heads of 128: 64 x 90 to 8000 1 / 2 / 4 / 8 72 / 68 / 67 / 72
// (in the sequences' order 72 / 71 / 72 / 76), of 8000 107 / 122 / 118 / 131; 32 x 100 to 8000 1 / 2 / 4 / 8 62 / 49 / 38 / 40;
// 64 x 90 to 4000 1 / 2 / 3 / 4 42 / 39 / 42 / 41; 16 x 90 to 20000 4 / 6 / 8 / 12 59 / 47 / 45 / 46; 16 x 4000 1 / 2 / 4 / 8 31 /
// 24 / 22.4 / 26; 100 x 90 to 8000 1 / 2 / 4 102 / 111 / 108; 4 x 2000 1 / 2 / 4 / 8 16 / 13.6 / 11 / 9.7; 1 x 2000 1 / 4 / 8 16 /
// 10.5 / 9.2; 1 x 30000 8 / 16 / 32 33 / 22.5 / 18; 8 x 1000 1 / 2 / 4 10.4 / 11.1 / 10.0; 4 heads of 64: 64 x 90 to 8000 1 / 2 /
// 4 / 8 39 / 33 / 31 / 35.
// Shared tiles (a workgroup to a CU): one to a CU where there are fewer, half as many again for several sequences; where
// they do not fill whole rounds, long contexts take the splits whose rounds come out best, of 4000 tokens or more, since a
// part of 256 rows is 130 KB.  8 x 100 x 300 to 8000 1 / 2 / 3 / 4 237 / 138 / 106 / 150; 16 x 40 x 1000 to 6000 1 / 2 / 3 / 4 179 /
// 107 / 91 / 116; 4 x 700 x 1100 to 4100 1 / 2 122 / 161; 1 x 1900 x 6400 1 / 2 203 / 240; 1 x 64 x 16000 1 / 8 / 16 / 32 470 /
// 75 / 49 / 60; 16 heads of 64: 2 x 128 x 6000 1 / 4 / 6 / 8 113 / 41 / 33 / 46; 1 x 3000 x 16000 1 / 2 / 3 / 4 / 6 350 / 357 / 338 /
// 301 / 318.
static KvAttnPlan kv4_attn_plan(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t D, int64_t max_q,
                                int64_t max_ctx, size_t scratch) {
  KvAttnPlan pl;
  const int64_t group = heads / kv_heads, rows = group * std::min(max_q, tokens);
  if (rows > 64) pl.tile = true, pl.rb = 256;
  else if (rows > 16) pl.nq = 2, pl.rb = 32;
  pl.blocks = tokens * group / pl.rb + batch;
  const int64_t there = std::max<int64_t>(1, std::min(pl.blocks, batch * cdiv(std::max<int64_t>(rows, 1), pl.rb)));
  pl.walk = batch > kDense ? pl.blocks : there;
  const int64_t units = pl.blocks * kv_heads, cus = device_cu_count(), step = pl.tile ? 64 : 256;
  const int64_t busy = there * kv_heads;  // workgroups with work, unsplit
  int64_t splits = 1;
  if (pl.tile) {
    splits = std::max<int64_t>(1, std::min((batch > 1 && 2 * busy >= cus ? 3 : 2) * cus / (2 * busy), max_ctx / (busy < 32 ? 1024 : 768)));
    for (int64_t n = 2; n <= 8 && max_ctx / n >= 4000; ++n)  // rounds of workgroups to a part
      if (2 * busy > cus && cdiv(busy * n, cus) * splits < cdiv(busy * splits, cus) * n) splits = n;
  } else {
    const int64_t least = busy <= 64 ? 256 : 512;
    if (max_ctx > 2 * least) splits = std::min((busy < 32 ? cus : 2 * cus) / busy, cdiv(max_ctx, least));
    if (batch > 1) splits = std::max({splits, std::min((4 * cus + busy / 2) / busy, max_ctx / 1024), max_ctx / 8192});
  }
  // a launch has less than 2^31 threads (the limit of rows leaves room for four splits at least)
  splits = std::max<int64_t>(1, std::min(splits, ((int64_t{1} << 31) / (pl.tile ? 512 : 256) - 1) / units));
  auto size = [&](int64_t n) { return n > 1 ? static_cast<size_t>(units) * n * pl.rb * (D + 2) * 4 : 0; };
  auto cut = [&](int64_t n) {
    pl.chunk = static_cast<int>(cdiv(cdiv(std::max<int64_t>(max_ctx, 1), n), step) * step);
    pl.splits = static_cast<int>(cdiv(std::max<int64_t>(max_ctx, 1), pl.chunk));
    pl.bytes = size(pl.splits);
  };
  cut(splits);
  pl.most = size(splits);
  if (pl.bytes > scratch)  // as many parts as it holds
    cut(std::max<int64_t>(1, static_cast<int64_t>(scratch / (static_cast<size_t>(units) * pl.rb * (D + 2) * 4))));
  return pl;
}

template <int D, int NQ>
static void launch_kv4_attn(const KvAttnPlan &pl, const Kv4AttnArgs &p, hipStream_t s) {
  constexpr int RB = 16 * NQ;
  const int64_t units = pl.blocks * p.kv_heads, rows = static_cast<int64_t>(p.tokens) * p.heads;
  hipLaunchKernelGGL((kv4_attn<D, NQ>), dim3(static_cast<unsigned>(units * pl.splits)), dim3(256), 0, s, p);
  if (pl.splits > 1)
    hipLaunchKernelGGL((kv_attn_combine<D, RB>), dim3(static_cast<unsigned>(cdiv(rows, 4))), dim3(256), 0, s, p);
}

template <int D>
static void launch_kv4_attn(const KvAttnPlan &pl, const Kv4AttnArgs &p, hipStream_t s) {
  if (pl.tile) {
    const int64_t units = pl.blocks * p.kv_heads, rows = static_cast<int64_t>(p.tokens) * p.heads;
    hipLaunchKernelGGL(kv4_attn_tile<D>, dim3(static_cast<unsigned>(units * pl.splits)), dim3(512), 0, s, p);
    if (pl.splits > 1)
      hipLaunchKernelGGL((kv_attn_combine<D, 256>), dim3(static_cast<unsigned>(cdiv(rows, 4))), dim3(256), 0, s, p);
  } else if (pl.nq == 2) launch_kv4_attn<D, 2>(pl, p, s);
  else launch_kv4_attn<D, 1>(pl, p, s);
}

}  // namespace teeny

using namespace teeny;

extern "C" {

teeny_status teeny_kv4_cache_attention(const void *q, const int8_t *k_cache, const int8_t *v_cache, const void *k_scale,
                                       const void *v_scale, const int32_t *block_table, const int32_t *context_lens,
                                       const int32_t *q_starts, void *o, float *l, int64_t n_tokens, int64_t batch,
                                       int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t num_pages,
                                       int64_t page_size, int64_t max_pages, int64_t max_q_len, int64_t max_context,
                                       int64_t q_stride, float softmax_scale, int32_t causal, teeny_stream stream) {
  const char *nm = "kv4_cache_attention";
  Kv4AttnArgs p{};
  KvAttnPlan pl;
  teeny_status st = kv_attn_open(nm, kv4_attn_plan, q, k_cache, v_cache, k_scale, v_scale, block_table, context_lens,
                                 q_starts, o, l, n_tokens, batch, q_heads, kv_heads, head_dim, num_pages, page_size,
                                 max_pages, max_q_len, max_context, q_stride, softmax_scale, causal, stream, p, pl);
  if (st != TEENY_OK || pl.blocks == 0) return st;
  TEENY_REQUIRE(aligned(k_scale, 4) && aligned(v_scale, 4), TEENY_ERR_MISALIGNED,
                "kv4_cache_attention: 4-byte aligned scales");
  p.ks = static_cast<const bf16 *>(k_scale);
  p.vs = static_cast<const bf16 *>(v_scale);
  p.sorted = !pl.tile && batch > 1 && batch <= 64 && pl.walk * pl.splits * kv_heads > 2 * device_cu_count();
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_dim == 64) launch_kv4_attn<64>(pl, p, s);
  else launch_kv4_attn<128>(pl, p, s);
  return after_launch(nm, s);
}

teeny_status teeny_kv4_cache_attention_workspace_size(int64_t n_tokens, int64_t batch, int64_t q_heads, int64_t kv_heads,
                                                      int64_t head_dim, int64_t max_q_len, int64_t max_context,
                                                      size_t *bytes) {
  return kv_attn_workspace("kv4_cache_attention_workspace_size", kv4_attn_plan, n_tokens, batch, q_heads, kv_heads, head_dim,
                           max_q_len, max_context, bytes);
}

}  // extern "C"
