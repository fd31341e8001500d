// Attention over the 8-bit paged K/V cache (kv_cache.hip), bf16 queries.
//
//   s = softmax_scale ks[page] (q . kq),  o = sum softmax(s) vs[page] vq
//
// for ragged batches: sequence b's queries are rows q_starts[b] ..
// q_starts[b + 1] - 1 of q [tokens, q_heads, D], the last tokens of its
// context.  No counterpart in the reference (flash_attn2.rs:52-158 reads
// dense K and V); grouped heads as teeny_attention_forward.
//
// Bound: for few queries by reading the cache once, for many by the products.
// The query rows that share a K/V head (its query heads times the sequence's
// queries) are the columns of v_mfma_f32_16x16x32_bf16: S^T = K Q^T, then
// O^T += V^T P^T.  A wave takes 64 tokens a time, 16 to each of its four lane
// groups: the score tiles' rows are dealt out so that lane group g's results
// are tokens 16 g .. 16 g + 15 of one query, which is one page (pages are
// whole multiples of 16): one K scale and one V scale per lane and round, and
// the probabilities are the next product's operand in the registers they were
// made in.  K's rows and V^T's rows then come straight from memory, 16 bytes
// a lane in whole 64-byte pieces, each byte to one lane: no LDS and no barrier
// in the loop.  Codes go to bf16 (exact) in registers, scales are applied in
// fp32: K's to the scores, V's to the probability before its rounding to bf16
// (the one rounding on the way, since the second product's operands are bf16: two
// bf16 parts would double that product; the row sum takes the unrounded
// probability).  It takes the rms error against 64 bits from 0.0017, the output's
// own rounding, to 0.0023.
// 64 contexts of 90 to 8000 tokens, 8 K/V heads of 128 and one query each, take
// 112 us (532 MB, 0.94 of the copy rate); one of 2000 tokens 10 us, where a wave's
// round of dependent work is 1.9 us and every load is waited for.
#include "mfma.hpp"

namespace teeny {

int kv_page_shift(int64_t page_size);

struct KvAttnArgs {
  const bf16 *q;
  int64_t q_stride;
  const int8_t *kc, *vc;
  const float *ks, *vs;
  const int32_t *table, *ctx, *starts;
  bf16 *o;
  float *l;
  float *part;      // [unit][split][row][D] fp32, then (at ml_off) [unit][split][row][2]; null: one split
  int64_t ml_off;
  int batch, tokens, heads, kv_heads, group, pages, shift, width;
  int blocks;       // row blocks of a head, over all sequences, at most
  int walk;         // of these, as many as the caller's lengths stand for
  int splits, chunk;  // chunk: tokens per split (a multiple of a workgroup's round)
  float scale_log2;
  int causal;
};

// A head's row block.  Its number, and so its place in the workspace, is
// floor(q_starts[b] group / RB) + b + its place in sequence b: distinct, and below
// tokens group / RB + batch, whatever the lengths.
struct KvRows {
  int b, row0, rows, len, first, ctx;  // rows: of the sequence and head; len: its queries; first: its first token's row
  template <int RB>
  __device__ __forceinline__ int number(const KvAttnArgs &p) const {
    return static_cast<int>(static_cast<int64_t>(first) * p.group / RB) + b + row0 / RB;
  }
};

// The last of up to n indexes from 0 on whose value, ascending, is not above x (0
// if there is none), 64 of them at a time.
template <typename F>
__device__ __forceinline__ int last_not_above(int n, int x, F value) {
  const int lane = threadIdx.x & 63;
  int at = 0;
  while (n > 1) {
    const int step = (n + 63) / 64;
    const uint64_t m = __ballot(lane * step < n && value(at + min(lane * step, n - 1)) <= x);
    const int k = m == 0 ? 0 : 63 - __builtin_clzll(m);
    at += k * step;
    n = min(step, n - k * step);
  }
  return at;
}

// Block u.  Up to kDense sequences: the u-th that there is, in the order of the
// sequences; the blocks beyond are none.  More of them: the one numbered u, which
// takes three loads for 4096 sequences where counting takes 64 (one token each for
// 4000 sequences of 20 to 60: 198 / 44 us; for 1024 of 100, 8 heads of 128, 159 / 109).
constexpr int kDense = 256;

template <int RB>
__device__ __forceinline__ bool kv_rows(const KvAttnArgs &p, uint32_t u, KvRows &r) {
  const int lane = threadIdx.x & 63;
  auto start = [&](int i) { return min(max(p.starts ? p.starts[i] : i, 0), p.tokens); };
  if (p.batch > kDense) {
    r.b = last_not_above(p.batch, u, [&](int i) { return static_cast<int>(static_cast<int64_t>(start(i)) * p.group / RB) + i; });
    r.first = start(r.b);
    r.len = start(r.b + 1) - r.first;
    r.rows = r.len * p.group;
    r.row0 = 0;
    r.row0 = (static_cast<int>(u) - r.number<RB>(p)) * RB;
    r.ctx = min(max(p.ctx[r.b], 0), p.width << p.shift);
    return r.len > 0 && r.row0 >= 0 && r.row0 < r.rows;
  }
  uint32_t before = 0;
  for (int i = 0; i < p.batch; i += 64) {
    const int b = min(i + lane, p.batch - 1), first = start(b), len = start(b + 1) - first, ctx = p.ctx[b];
    const uint32_t nb = i + lane < p.batch && len > 0 ? (len * p.group + RB - 1) / RB : 0, upto = wave_scan(nb);
    const uint32_t here = __builtin_amdgcn_readlane(upto, 63);
    if (u - before < here) {
      const int at = __builtin_ctzll(__ballot(upto > u - before));
      auto from = [&](int v) { return __builtin_amdgcn_readlane(v, at); };
      r.b = i + at;
      r.first = from(first);
      r.len = from(len);
      r.rows = r.len * p.group;
      r.row0 = static_cast<int>(u - before - from(upto - nb)) * RB;
      r.ctx = min(max(from(ctx), 0), p.width << p.shift);
      return true;
    }
    before += here;
  }
  return false;
}

// The same blocks in order of their work, the longest first, for up to 64
// sequences: a later, longer block would run on alone when the others are done.
// Lane b counts its sequence's blocks that see more than T tokens; the count over
// all sequences is above u for T up to the block's own, found by bisection.
template <int RB>
__device__ __forceinline__ bool kv_rows_sorted(const KvAttnArgs &p, int u, KvRows &r) {
  if (p.batch > 64) return kv_rows<RB>(p, u, r);
  const int lane = threadIdx.x & 63, b = min(lane, p.batch - 1);
  auto start = [&](int i) { return min(max(p.starts ? p.starts[i] : i, 0), p.tokens); };
  const int first = start(b), len = lane < p.batch ? max(start(b + 1) - first, 0) : 0;
  const int rows = len * p.group, nb = (rows + RB - 1) / RB;
  const int ctx = min(max(p.ctx[b], 0), p.width << p.shift);
  // blocks (from the last one down) whose last row sees more than 64 tau - 1 tokens
  auto count = [&](int tau) -> uint32_t {
    if (tau == 0) return nb;
    const int t = 64 * tau - 1;
    if (ctx <= t) return 0;
    if (!p.causal) return nb;
    // block nb - 1 - i, i > 0, ends with row (nb - i) RB - 1, whose query sees ctx - len + 1 + row / group tokens
    const int64_t need = (static_cast<int64_t>(t) - ctx + len) * p.group + 1;
    return need <= 1 ? nb : max(1, nb - static_cast<int>((need + RB - 1) / RB) + 1);
  };
  auto total = [&](uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(wave_scan(v)), 63)); };
  if (total(nb) <= static_cast<uint32_t>(u)) return false;
  int lo = 0, hi = (p.width << p.shift) / 64 + 1;  // total(count(lo)) > u >= total(count(hi)) = 0
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (total(count(mid)) > static_cast<uint32_t>(u)) lo = mid;
    else hi = mid;
  }
  const uint32_t above = count(hi), here = count(lo) - above, upto = wave_scan(here);
  const uint32_t at = u - total(above);
  const int owner = __builtin_ctzll(__ballot(upto > at));
  auto from = [&](int v) { return __builtin_amdgcn_readlane(v, owner); };
  r.b = owner;
  r.first = from(first);
  r.len = from(len);
  r.rows = from(rows);
  r.ctx = from(ctx);
  r.row0 = (from(nb) - 1 - static_cast<int>(from(above) + at - (from(upto) - from(here)))) * RB;
  return true;
}

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Eight int8 codes as bf16.  The words are opaque here, or the compiler carries
// a loop's loads on as single bytes, a register each.
__device__ __forceinline__ bf16x8 codes8(uint32_t lo, uint32_t hi) {
  asm("" : "+v"(lo), "+v"(hi));
  bf16x8 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t word = (j < 2 ? lo : hi) >> (16 * (j & 1));
    const bf16x2 pr = cvt_pk_bf16(static_cast<float>(static_cast<int8_t>(word & 0xffu)),
                                  static_cast<float>(static_cast<int8_t>((word >> 8) & 0xffu)));
    r[2 * j] = pr[0];
    r[2 * j + 1] = pr[1];
  }
  return r;
}

// The same value in the four lanes l % 16, l % 16 + 16, ..: their maximum or sum.
template <typename F>
__device__ __forceinline__ float over_groups(float v, F f) {
  v = f(v, __shfl_xor(v, 16, 64));
  return f(v, __shfl_xor(v, 32, 64));
}

// NQ: 16-row column blocks; the four waves share out the tokens, 64 a time.
template <int D, int NQ>
__global__ __launch_bounds__(256, NQ == 1 && D == 64 ? 4 : 2) void kv_attn(KvAttnArgs p) {
  constexpr int WK = 4, WROWS = 16 * NQ, RB = WROWS;
  constexpr int NC = D / 32, ND = D / 16, NL = D / 64;  // k-steps of the scores, d blocks, 16-byte pieces of a K row
  constexpr int LD = D + 4;
  __shared__ __attribute__((aligned(16))) float red[WK * WROWS * LD];
  __shared__ float ml[2][WK][WROWS];
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  // the blocks that the caller's lengths stand for come first, then those that there may be beyond, mostly none
  const int per_block = p.splits * p.kv_heads, first = p.walk * per_block;
  const bool beyond = static_cast<int>(blockIdx.x) >= first;
  const int id = beyond ? blockIdx.x - first : xcd_remap(blockIdx.x, first), of = beyond ? p.blocks - p.walk : p.walk;
  const int head = id / (p.splits * of), in_head = id - head * (p.splits * of), split = in_head / of;
  KvRows r;
  if (!kv_rows<RB>(p, in_head - split * of + (beyond ? p.walk : 0), r)) return;
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
  u32x4 kr[4][NL], vr[ND];
  float ksc = 0.0f, vsc = 0.0f;
  bool none = false;
  auto load_k = [&](int t0, Pages pg) {
    const int64_t at = (static_cast<int64_t>(max(pg.k, 0)) * p.kv_heads + head) << p.shift;
    const int8_t *src = p.kc + (at + ((t0 + 16 * (c >> 2)) & page_mask) + (c & 3)) * D + 16 * g;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < NL; ++j) kr[i][j] = *reinterpret_cast<const u32x4 *>(src + 4 * i * D + 64 * j);
  };
  auto load_v = [&](int t0, Pages pg) {
    const int64_t unit_at = static_cast<int64_t>(max(pg.v, 0)) * p.kv_heads + head;
    const int8_t *src = p.vc + (((unit_at * D + c) << p.shift) + ((t0 + 16 * g) & page_mask));
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      vr[d] = *reinterpret_cast<const u32x4 *>(src);
      src += 16 << p.shift;
    }
    ksc = p.ks[unit_at];
    vsc = p.vs[unit_at];
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

  const float sc0 = fabsf(p.scale_log2);
  const uint32_t qsign = p.scale_log2 < 0.0f ? 0x80008000u : 0u;  // a negative scale's sign goes to Q
  bf16x8 qf[NQ][NC];
  int vis[NQ];
  int64_t out_row[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int i = min(r.row0 + 16 * n + c, r.rows - 1), t = i / p.group;
    vis[n] = p.causal ? min(max(r.ctx - r.len + 1 + t, 0), r.ctx) : r.ctx;
    const int h = head * p.group + i - t * p.group;
    out_row[n] = static_cast<int64_t>(r.first + t) * p.heads + h;
    const bf16 *at = p.q + (r.first + t) * p.q_stride + h * D;
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      u32x4 raw = *reinterpret_cast<const u32x4 *>(at + (j >> 1) * 64 + g * 16 + (j & 1) * 8);
      raw ^= qsign;
      qf[n][j] = __builtin_bit_cast(bf16x8, raw);
    }
  }
  const int all_see = seen(r.row0);  // all rows see the tokens below it

  f32x4 acc[NQ][ND];
  float m_run[NQ], l_run[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    m_run[n] = -INFINITY;
    l_run[n] = 0.0f;
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[n][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
#pragma unroll 1
  for (; t0 < ke; t0 += STEP) {
    f32x4 s[NQ][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) s[n][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        const bf16x8 a = codes8(kr[i][j >> 1][2 * (j & 1)], kr[i][j >> 1][2 * (j & 1) + 1]);
#pragma unroll
        for (int n = 0; n < NQ; ++n) s[n][i] = mfma16(a, qf[n][j], s[n][i]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    const bool more = t0 + STEP < ke;
    // at least FLT_MIN, so that a masked -inf gives p = 0 under a zero scale too; NaN stays
    const float sc = __builtin_elementwise_maximum(sc0 * ksc, 1.17549435e-38f), vmul = vsc;
    const bool hidden = none;
    if (more) load_k(t0 + STEP, pg);
    const bool masks = t0 + 64 > all_see || __any(hidden);
    const int at = t0 + 16 * g;  // the lane's first token
    bf16x8 pb[NQ][2];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float scn = sc;
      if (masks) {
        if (hidden || at >= vis[n]) scn = 1.17549435e-38f;  // the scale of a page that the row does not see may be anything
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (hidden || at + i >= vis[n]) s[n][i >> 2][i & 3] = -INFINITY;
      }
      float mx = s[n][0][0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = __builtin_elementwise_maximum(mx, s[n][i >> 2][i & 3]);
      mx = over_groups(mx * scn, [](float a, float b) { return __builtin_elementwise_maximum(a, b); });
      if (__any(mx > m_run[n] + 8.0f)) {  // rescaled rarely: p <= 2^8
        const float m_new = fmaxf(m_run[n], mx);
        const float alpha = __builtin_amdgcn_exp2f(m_run[n] - (m_new == -INFINITY ? 0.0f : m_new));
        l_run[n] *= alpha;
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[n][d] *= alpha;
        m_run[n] = m_new;
      }
      const float neg_m = m_run[n] == -INFINITY ? 0.0f : -m_run[n];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][i >> 2][i & 3], scn, neg_m));
        l_run[n] += e;
        s[n][i >> 2][i & 3] = masks && (hidden || at + i >= vis[n]) ? 0.0f : e * vmul;  // a hidden token's V scale may be anything
      }
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const bf16x2 pr = cvt_pk_bf16(s[n][i >> 2][i & 3], s[n][i >> 2][(i & 3) + 1]);
        pb[n][i >> 3][i & 7] = pr[0];
        pb[n][i >> 3][(i & 7) + 1] = pr[1];
      }
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bf16x8 a = codes8(vr[d][2 * h], vr[d][2 * h + 1]);
#pragma unroll
        for (int n = 0; n < NQ; ++n) acc[n][d] = mfma16(a, pb[n][h], acc[n][d]);
      }
      __builtin_amdgcn_sched_barrier(0);
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
    const float mul = __builtin_amdgcn_exp2f(m_run[n] - ref) * (whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f);
#pragma unroll
    for (int d = 0; d < ND; ++d)
      *reinterpret_cast<f32x4 *>(red + (w * WROWS + at) * LD + 16 * d + 4 * g) = acc[n][d] * mul;
    if (w == 0 && g == 0 && r.row0 + at < r.rows) {
      if (!whole) {
        p.part[p.ml_off + (slot + at) * 2] = m;
        p.part[p.ml_off + (slot + at) * 2 + 1] = l;
      } else if (p.l != nullptr) {
        p.l[out_row[n]] = (m + log2f(l)) * 0.6931471805599453f;
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

// Many query rows (prompts in pieces): bound by the products, and next by
// turning codes into operands, which in kv_attn every wave does for itself.
// Here a workgroup of four waves, 32 rows each, turns a tile of 64 tokens once:
// its lanes read 16 codes each of K and of V per D / 64, and write the bf16
// operands of v_mfma_f32_32x32x16_bf16 to LDS in the order in which lanes take
// them up, 1 KiB a product, so that writes and reads are without conflicts.  The
// codes of the tile after next are in flight meanwhile; one barrier a tile, two
// tiles in LDS, two workgroups on a CU, whose products and exponentials overlap.
// Rows of the scores are dealt out as in kv_attn: lane half g's results of a
// block of 32 tokens are tokens 16 g .. 16 g + 15 of one query, one page.
// 700 queries of 32 heads of 128 for each of four contexts of 1100 to 4100 tokens:
// 144 us (319 with kv_attn), 647 TFLOP/s; 823 where contexts are of one length.
// (Calls in a row; one after a pause takes 161.)
template <int D>
__global__ __launch_bounds__(256, 2) void kv_attn_tile(KvAttnArgs p) {
  constexpr int RB = 128, NS = D / 16, ND = D / 32, NU = D / 64, FR = 2 * NS + 4 * ND;
  __shared__ __attribute__((aligned(16))) u32x4 frag[2][FR * 64];  // K [block][step], then V [d block][block][half]
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

  const float sc0 = fabsf(p.scale_log2);
  const uint32_t qsign = p.scale_log2 < 0.0f ? 0x80008000u : 0u;
  const int my = min(base + c, r.rows - 1), qt = my / p.group, qh = head * p.group + my - qt * p.group;
  const int64_t out_row = static_cast<int64_t>(r.first + qt) * p.heads + qh;
  const int vis = seen(my), all_see = seen(min(base, r.rows - 1));
  const int w_end = base < r.rows ? min(ke, seen(min(base + 32, r.rows) - 1)) : 0;
  bf16x8 qf[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    u32x4 raw = *reinterpret_cast<const u32x4 *>(p.q + (r.first + qt) * p.q_stride + qh * D + (i >> 1) * 32 + g * 16 + (i & 1) * 8);
    raw ^= qsign;
    qf[i] = __builtin_bit_cast(bf16x8, raw);
  }
  f32x16 acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) acc[d] = zero16();
  float m_run = -INFINITY, l_run = 0.0f;

  // The wave's share of a tile: K rows of block w / 2 (D = 128: 64 bytes of each row in two pieces), and V rows of
  // d block w, tokens of both blocks (D = 64: of d block w / 2 and block w % 2).  The four pages of a tile are one
  // load for the wave; what follows from them is the same for all lanes and is worked out in scalar registers.
  const int32_t *row = p.table + static_cast<int64_t>(r.b) * p.width;
  const int page_mask = (1 << p.shift) - 1, wb = w >> 1;
  const bool k_odd = (c >> 2) & 1, g_odd = g;
  const int k_lane = (4 * (c >> 3) + (c & 3)) * D + 16 * g + (D == 128 ? 64 : 32) * (w & 1);
  const int v_lane = (32 * (D == 128 ? w : wb) + c) << p.shift;
  auto v_block = [&](int i) { return D == 128 ? i : w & 1; };
  // lane l: the page of tokens 16 (l % 4) .. of a tile
  auto load_pages = [&](int t0) { return row[min(t0 + 16 * (lane & 3), k_end - 1) >> p.shift]; };
  u32x4 kr[NU], vr[NU];
  float ks_next[2], vs_next[2];
  bool none_next[2];
  auto load_codes = [&](int t0, int pg) {
    uint32_t at[4];  // (page, head) index: below 2^29
    int in[4];       // offset in the page
    bool there[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int page = __builtin_amdgcn_readlane(pg, j), t = t0 + 16 * j;
      there[j] = page >= 0 && page < p.pages && t < ke;
      at[j] = static_cast<uint32_t>(there[j] ? page : 0) * p.kv_heads + head;
      in[j] = t & page_mask;
    }
    auto pick = [&](bool odd, int64_t x, int64_t y) { return odd ? y : x; };
    auto k_off = [&](int j) { return ((static_cast<int64_t>(at[j]) << p.shift) + in[j]) * D; };
    auto v_off = [&](int j) { return (static_cast<int64_t>(at[j]) * D << p.shift) + in[j]; };
    const int8_t *k_src = p.kc + (pick(k_odd, wb ? k_off(2) : k_off(0), wb ? k_off(3) : k_off(1)) + k_lane);
#pragma unroll
    for (int i = 0; i < NU; ++i) kr[i] = *reinterpret_cast<const u32x4 *>(k_src + 32 * i);
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int v = v_block(i);
      vr[i] = *reinterpret_cast<const u32x4 *>(p.vc + (pick(g_odd, v ? v_off(2) : v_off(0), v ? v_off(3) : v_off(1)) + v_lane));
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const uint32_t i = g_odd ? at[2 * b + 1] : at[2 * b];
      ks_next[b] = p.ks[i];
      vs_next[b] = p.vs[i];
      none_next[b] = g_odd ? !there[2 * b + 1] : !there[2 * b];
    }
  };
  auto turn = [&](u32x4 *to) {
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int step = 2 * (NU * (w & 1) + i), at = (w >> 1) * NS + step;
      to[at * 64 + lane] = __builtin_bit_cast(u32x4, codes8(kr[i][0], kr[i][1]));
      to[(at + 1) * 64 + lane] = __builtin_bit_cast(u32x4, codes8(kr[i][2], kr[i][3]));
    }
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int at = 2 * NS + ((D == 128 ? w : w >> 1) * 2 + v_block(i)) * 2;
      to[at * 64 + lane] = __builtin_bit_cast(u32x4, codes8(vr[i][0], vr[i][1]));
      to[(at + 1) * 64 + lane] = __builtin_bit_cast(u32x4, codes8(vr[i][2], vr[i][3]));
    }
  };

  int pg = 0, buf = 0;
  float ksc[2], vsc[2];
  bool none[2];
  auto take = [&]() {
#pragma unroll
    for (int b = 0; b < 2; ++b) ksc[b] = ks_next[b], vsc[b] = vs_next[b], none[b] = none_next[b];
  };
  if (kb < ke) {
    pg = load_pages(kb);
    load_codes(kb, pg);
    pg = load_pages(kb + 64);
    turn(frag[0]);
    take();
    if (kb + 64 < ke) {
      load_codes(kb + 64, pg);
      pg = load_pages(kb + 128);
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int t0 = kb; t0 < ke; t0 += 64) {
    const u32x4 *now = frag[buf];
    const float sc1[2] = {__builtin_elementwise_maximum(sc0 * ksc[0], 1.17549435e-38f),
                          __builtin_elementwise_maximum(sc0 * ksc[1], 1.17549435e-38f)};
    float vm[2] = {vsc[0], vsc[1]};
    const bool hidden[2] = {none[0], none[1]};
    if (t0 + 64 < ke) {
      turn(frag[buf ^ 1]);
      take();
      if (t0 + 128 < ke) {
        load_codes(t0 + 128, pg);
        pg = load_pages(t0 + 192);
      }
    }
    if (t0 < w_end) {
      // operands are read LA products ahead, V's first ones before the exponentials; the order is kept as written
      constexpr int LA = 4, W = LA + 1;
      u32x4 win[W];
      auto read = [&](int i) __attribute__((always_inline)) {
        const int j = i - 2 * NS;  // scores: both blocks in turn; outputs: the d blocks in turn
        const int at = i < 2 * NS ? (i & 1) * NS + (i >> 1) : 2 * NS + (j % ND) * 4 + j / ND;
        win[i % W] = now[at * 64 + lane];
      };
#pragma unroll
      for (int i = 0; i < LA; ++i) read(i);
      f32x16 s[2] = {zero16(), zero16()};
#pragma unroll
      for (int i = 0; i < 2 * NS; ++i) {
        read(i + LA);
        s[i & 1] = mfma32x32x16(__builtin_bit_cast(bf16x8, win[i % W]), qf[i >> 1], s[i & 1]);
        __builtin_amdgcn_sched_barrier(0);
      }
      const bool masks = t0 + 64 > all_see || __any(hidden[0] || hidden[1]);
      float sc[2] = {sc1[0], sc1[1]};
      if (masks) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int at = t0 + 32 * b + 16 * g;
          if (hidden[b] || at >= vis) sc[b] = 1.17549435e-38f;  // the scale of a page that the row does not see may be anything
#pragma unroll
          for (int v = 0; v < 16; ++v)
            if (hidden[b] || at + v >= vis) s[b][v] = -INFINITY;
        }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        float x = s[b][0];
#pragma unroll
        for (int v = 1; v < 16; ++v) x = __builtin_elementwise_maximum(x, s[b][v]);
        mx = __builtin_elementwise_maximum(mx, x * sc[b]);
      }
      mx = __builtin_elementwise_maximum(mx, __shfl_xor(mx, 32, 64));
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
      // p vs[page] as exp2(s - m + log2 vs), where every scale of the wave has a logarithm (one multiplication less a
      // score; the sum is divided by the scale again); what is hidden takes the scale 1
      bool plain = true;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        if (masks && (hidden[b] || t0 + 32 * b + 16 * g >= vis)) vm[b] = 1.0f;
        plain = plain && vm[b] > 1e-30f && vm[b] < 1e30f;
      }
      plain = __all(plain);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        if (plain) {
          const float off = neg_m + __builtin_amdgcn_logf(vm[b]);
          float sum = 0.0f;
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            s[b][v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][v], sc[b], off));
            sum += s[b][v];
          }
          l_run = __builtin_fmaf(sum, __builtin_amdgcn_rcpf(vm[b]), l_run);
        } else {
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][v], sc[b], neg_m));
            l_run += e;
            s[b][v] = e * vm[b];
          }
          if (masks) {  // a hidden token of a page that the row sees in part: its scale may be infinite
#pragma unroll
            for (int v = 0; v < 16; ++v)
              if (hidden[b] || t0 + 32 * b + 16 * g + v >= vis) s[b][v] = 0.0f;
          }
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
        acc[d] = mfma32x32x16(__builtin_bit_cast(bf16x8, win[i % W]), pb[bh >> 1][bh & 1], acc[d]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    buf ^= 1;
    __syncthreads();
  }
  l_run += __shfl_xor(l_run, 32, 64);
  if (base + c >= r.rows) return;
  const bool whole = p.part == nullptr || k_end <= p.chunk;  // no other split has a part of these rows
  const int64_t unit = static_cast<int64_t>(head) * p.blocks + r.number<RB>(p);
  const int64_t slot = (unit * p.splits + split) * RB + 32 * w + c;
  const float mul = whole ? (l_run == 0.0f ? 0.0f : 1.0f / l_run) : 1.0f;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int at = 32 * d + 8 * a + 4 * g;
      if (whole) {
        bf16x4 o4;
#pragma unroll
        for (int v = 0; v < 4; ++v) o4[v] = static_cast<bf16>(acc[d][4 * a + v] * mul);
        *reinterpret_cast<bf16x4 *>(p.o + out_row * D + at) = o4;
      } else {
        *reinterpret_cast<f32x4 *>(p.part + slot * D + at) = f32x4{acc[d][4 * a], acc[d][4 * a + 1], acc[d][4 * a + 2], acc[d][4 * a + 3]};
      }
    }
  if (g == 0 && !whole) {
    p.part[p.ml_off + slot * 2] = m_run;
    p.part[p.ml_off + slot * 2 + 1] = l_run;
  } else if (g == 0 && p.l != nullptr) {
    p.l[out_row] = (m_run + log2f(l_run)) * 0.6931471805599453f;
  }
}

// One wave per row of the output: the splits' parts, in split order.  2048 rows of
// up to three parts of 128 take 5 us, 32 rows of eight 3 us: mostly the launch.
template <int D, int RB>
__global__ __launch_bounds__(256) void kv_attn_combine(KvAttnArgs p) {
  constexpr int V = D / 64;
  typedef float fv __attribute__((ext_vector_type(V)));
  const int lane = threadIdx.x & 63;
  const uint32_t row = blockIdx.x * 4u + (threadIdx.x >> 6);  // below 2^31
  const int t = row / p.heads, h = static_cast<int>(row - static_cast<uint32_t>(t) * p.heads), head = h / p.group;
  if (t >= p.tokens) return;
  // the row's sequence, and its place among the sequence's rows
  auto start = [&](int i) { return min(max(p.starts ? p.starts[i] : i, 0), p.tokens); };
  const int b = last_not_above(p.batch, t, start), first = start(b), end = start(b + 1);
  if (t < first || t >= end) return;
  const int ctx = min(max(p.ctx[b], 0), p.width << p.shift);
  const int i = (t - first) * p.group + h - head * p.group, len = end - first;
  const int last = min(i / RB * RB + RB, len * p.group) - 1;
  const int k_end = p.causal ? min(max(ctx - len + 1 + last / p.group, 0), ctx) : ctx;
  if (k_end <= p.chunk) return;  // the one split that saw the row wrote its output
  const int n = min(p.splits, (k_end - 1) / p.chunk + 1);
  const int unit = head * p.blocks + static_cast<int>(static_cast<int64_t>(first) * p.group / RB) + b + i / RB;
  const int64_t slot = static_cast<int64_t>(unit) * p.splits * RB + i % RB;
  const float *ml = p.part + p.ml_off;
  float m = -INFINITY;
  for (int s = lane; s < n; s += 64) m = fmaxf(m, ml[(slot + static_cast<int64_t>(s) * RB) * 2]);
  m = wave_max(m);
  const float ref = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
  fv o = {};
  for (int s0 = 0; s0 < n; s0 += 64) {  // a lane's factor is of split s0 + lane
    float f = 0.0f, ls = 0.0f;
    if (s0 + lane < n) {
      const float *of = ml + (slot + static_cast<int64_t>(s0 + lane) * RB) * 2;
      f = __builtin_amdgcn_exp2f(of[0] - ref);
      ls = of[1] * f;
    }
    l += wave_sum(ls);
    const int here = min(n - s0, 64);
    const float *at = p.part + (slot + static_cast<int64_t>(s0) * RB) * D + lane * V;
    for (int s = 0; s < here; s += 8) {  // eight loads in flight; past the last split its part again, times 0
      fv x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = *reinterpret_cast<const fv *>(at + static_cast<int64_t>(min(s + j, here - 1)) * (RB * D));
#pragma unroll
      for (int j = 0; j < 8; ++j) o += x[j] * __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), s + j));
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int j = 0; j < V; ++j) p.o[static_cast<int64_t>(row) * D + lane * V + j] = static_cast<bf16>(o[j] * inv);
  if (p.l != nullptr && lane == 0) p.l[row] = (m + log2f(l)) * 0.6931471805599453f;
}

// ── which form, and how many splits ─────────────────────────────────────────
// Few rows take kv_attn, more than 64 a sequence the shared tiles.  kv_attn's
// splits give a workgroup one round of 256 tokens where they leave CUs free (a
// round is 1.9 us of dependent work, a row's other parts 0.04 us each), two rounds
// where the device is busier, from three rounds on; more workgroups than two to a
// CU (one where there are few: their parts count) only where contexts may differ
// much in length.  us by splits, 8 K/V heads of 128, one query: 1 x 600 1 / 3 10.6
// / 9.9; 1 x 2000 1 / 4 / 8 20 / 12.5 / 10.7; 1 x 30000 16 / 32 / 64 28 / 21.7 /
// 23.3; 4 x 2000 4 / 8 13.4 / 12.1; 8 x 1000 1 / 2 / 4 14.4 / 13.7 / 12.3; 8 x 4000
// 4 / 6 / 8 20.9 / 22.4 / 20.4; 16 x 1000 1 / 2 / 4 14.6 / 15.8 / 15.4; 16 x 4000 2
// / 4 / 8 33 / 33 / 36; 32 x 2000 1 / 2 28.8 / 33.3, but 32 x 100 to 8000 1 / 2 / 3
// 83 / 71 / 65; 64 x 90 to 8000 1 / 2 / 3 / 4 116 / 126 / 112 / 117.  Several long
// contexts, which may differ, get a split for each 2560 tokens, so three from 7680
// on: 64 x 90 to 12000 1 / 3 / 4 / 5 172 / 162 / 167 / 164 (but 64 x 8000 187 / 195
// / 196 / 201), 16 x 90 to 20000 4 / 5 / 7 / 10 86 / 79 / 94 / 86, 4 x 1000 to
// 40000 6 / 8 / 10 / 15 59 / 48 / 55 / 43.  Two do not pay where the unsplit call
// just fills two workgroups a CU (1 / 2 / 3: 64 x 90 to 5200 80 / 87 / 82, to 6400
// 96 / 104 / 96, to 7600 113 / 120 / 112, 64 x 6400 151 / 158 / 160, 56 x 90 to
// 6400 90 / 95 / 90), but with fewer and with more (90 to 6400: 48 x 86 / 85 / 84,
// 80 x 126 / 121 / 119, 96 x 150 / 144 / 139, 128 x 184 / 177 / 177; 200 x 90 to
// 5200 216 / 219 / 225).  One sequence alone has nothing to even out: 1 x 30000, 64
// heads, 8 / 11 96 / 110, 1 x 60000, 32 heads, 16 / 23 96 / 117.  Shared tiles: 1 x
// 64 queries x 16000 1 / 8 / 16 / 32 488 / 76 / 60 / 52; 2 x 128 x 6000, 16 heads
// of 64, 1 / 4 / 8 / 16 145 / 49 / 39 / 46; 8 x 100 x 300 to 8000 1 / 2 / 3 / 4 242
// / 180 / 139 / 160; 4 x 700 x 1100 to 4100 1 / 2 160 / 193; with the split for
// 2560 tokens 15 x 100 x 300 to 6400 1 / 2 / 3 197 / 167 / 183 (of 6400 255 / 286 /
// 290), 1 x 3000 x 16000, 16 heads of 64, 1 / 3 / 6 / 10 453 / 375 / 363 / 383, 1 x
// 1900 x 6400 1 / 2 223 / 255, 1 x 1500 x 8000 1 / 3 281 / 274.  Several sequences
// on a busy device get half as many again, since contexts seldom are of one length:
// 16 x 40 x 1000 to 6000 2 / 3 / 4 133 / 101 / 125, of 4000 104 / 116 / 110; 20 x
// 40 x 300 to 4000 1 / 2 125 / 97, of 2000 88 / 98.
struct KvAttnPlan {
  bool tile = false;
  int nq = 1, rb = 16;
  int64_t blocks = 0, walk = 0;  // row blocks of a head at most; as the lengths have it
  int splits = 1, chunk = 0;
  size_t bytes = 0, most = 0;  // of workspace: used; enough for this and any smaller max_context
};

static KvAttnPlan kv_attn_plan(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t D,
                               int64_t max_q, int64_t max_ctx, size_t scratch) {
  KvAttnPlan pl;
  const int64_t group = heads / kv_heads, rows = group * std::min(max_q, tokens);
  if (rows > 64) pl.tile = true, pl.rb = 128;
  else if (rows > 16) pl.nq = 2, pl.rb = 32;
  pl.blocks = tokens * group / pl.rb + batch;
  const int64_t there = std::max<int64_t>(1, std::min(pl.blocks, batch * cdiv(std::max<int64_t>(rows, 1), pl.rb)));
  pl.walk = batch > kDense ? pl.blocks : there;
  const int64_t units = pl.blocks * kv_heads, cus = device_cu_count(), step = pl.tile ? 64 : 256;
  const int64_t busy = there * kv_heads;  // workgroups with work, unsplit
  const int64_t least = pl.tile ? (busy < 32 ? 256 : 768) : busy <= 64 ? 256 : 512;
  int64_t splits = 1;
  if (pl.tile) splits = std::min((batch > 1 && 2 * busy > cus ? 3 : 2) * cus / busy, max_ctx / least);
  else if (max_ctx > 2 * least) splits = std::min((busy < 32 ? cus : 2 * cus) / busy, cdiv(max_ctx, least));
  const int64_t pieces = max_ctx / 2560;
  const bool two = pl.tile || 5 * busy <= 8 * cus || busy > 2 * cus;  // whether two splits may pay
  if (pl.tile ? busy < 2 * cus : busy >= 32 && batch > 1 && (pieces > 2 || two)) splits = std::max(splits, pieces);
  // a launch has less than 2^31 threads (the limit of rows leaves room for four splits at least)
  splits = std::max<int64_t>(1, std::min(splits, ((int64_t{1} << 31) / 256 - 1) / units));
  auto size = [&](int64_t n) { return n > 1 ? static_cast<size_t>(units) * n * pl.rb * (D + 2) * 4 : 0; };
  auto cut = [&](int64_t n) {
    pl.chunk = static_cast<int>(cdiv(cdiv(std::max<int64_t>(max_ctx, 1), n), step) * step);
    pl.splits = static_cast<int>(cdiv(std::max<int64_t>(max_ctx, 1), pl.chunk));
    pl.bytes = size(pl.splits);
  };
  cut(splits);
  pl.most = size(splits);
  if (pl.bytes > scratch) {  // as many parts as it holds
    const int64_t fit = static_cast<int64_t>(scratch / (static_cast<size_t>(units) * pl.rb * (D + 2) * 4));
    cut(std::max<int64_t>(1, fit == 2 && !two ? 1 : fit));
  }
  return pl;
}

template <int D, int NQ>
static void launch_kv_attn(const KvAttnPlan &pl, const KvAttnArgs &p, hipStream_t s) {
  constexpr int RB = 16 * NQ;
  const int64_t units = pl.blocks * p.kv_heads, rows = static_cast<int64_t>(p.tokens) * p.heads;
  hipLaunchKernelGGL((kv_attn<D, NQ>), dim3(static_cast<unsigned>(units * pl.splits)), dim3(256), 0, s, p);
  if (pl.splits > 1)
    hipLaunchKernelGGL((kv_attn_combine<D, RB>), dim3(static_cast<unsigned>(cdiv(rows, 4))), dim3(256), 0, s, p);
}

template <int D>
static void launch_kv_attn(const KvAttnPlan &pl, const KvAttnArgs &p, hipStream_t s) {
  if (pl.tile) {
    const int64_t units = pl.blocks * p.kv_heads, rows = static_cast<int64_t>(p.tokens) * p.heads;
    hipLaunchKernelGGL(kv_attn_tile<D>, dim3(static_cast<unsigned>(units * pl.splits)), dim3(256), 0, s, p);
    if (pl.splits > 1)
      hipLaunchKernelGGL((kv_attn_combine<D, 128>), dim3(static_cast<unsigned>(cdiv(rows, 4))), dim3(256), 0, s, p);
  }
  else if (pl.nq == 2) launch_kv_attn<D, 2>(pl, p, s);
  else launch_kv_attn<D, 1>(pl, p, s);
}

static teeny_status kv_attn_sizes(const char *nm, int64_t n_tokens, int64_t batch, int64_t q_heads, int64_t kv_heads,
                                  int64_t head_dim, int64_t max_q_len, int64_t max_context) {
  const std::string at = std::string(nm) + ": ";
  TEENY_REQUIRE(n_tokens >= 0 && batch >= 0 && q_heads >= 0 && kv_heads >= 0 && max_q_len >= 0 && max_context >= 0,
                TEENY_ERR_SHAPE_MISMATCH, at + "negative size");
  TEENY_REQUIRE(head_dim == 64 || head_dim == 128, TEENY_ERR_UNSUPPORTED, at + "head_dim must be 64 or 128");
  TEENY_REQUIRE(kv_heads > 0 ? q_heads % kv_heads == 0 : q_heads == 0, TEENY_ERR_SHAPE_MISMATCH,
                at + "q_heads must be a multiple of kv_heads");
  TEENY_REQUIRE(n_tokens <= 0x7fffffff && batch < 0x7fffffff && max_context <= 0x7fffffff - 4096 &&
                    q_heads <= 65535 && n_tokens * q_heads <= 0x7fffffff && batch * q_heads <= 0x7fffffff,
                TEENY_ERR_SHAPE_MISMATCH, at + "tokens * q_heads, batch * q_heads or max_context exceed 2^31-1");
  return TEENY_OK;
}

}  // namespace teeny

using namespace teeny;

extern "C" {

teeny_status teeny_kv_cache_attention(const void *q, const int8_t *k_cache, const int8_t *v_cache, const float *k_scale,
                                      const float *v_scale, const int32_t *block_table, const int32_t *context_lens,
                                      const int32_t *q_starts, void *o, float *l, int64_t n_tokens, int64_t batch,
                                      int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t num_pages,
                                      int64_t page_size, int64_t max_pages, int64_t max_q_len, int64_t max_context,
                                      int64_t q_stride, float softmax_scale, int32_t causal, teeny_stream stream) {
  const char *nm = "kv_cache_attention";
  teeny_status st = kv_attn_sizes(nm, n_tokens, batch, q_heads, kv_heads, head_dim, max_q_len, max_context);
  if (st != TEENY_OK) return st;
  const int shift = kv_page_shift(page_size);
  TEENY_REQUIRE(shift > 0, TEENY_ERR_UNSUPPORTED, "kv_cache_attention: page_size must be 16, 32, 64 or 128");
  TEENY_REQUIRE(num_pages >= 0 && max_pages >= 0 && num_pages <= 0x7fffffff / page_size &&
                    max_pages <= (0x7fffffff - 4096) / page_size,
                TEENY_ERR_SHAPE_MISMATCH, "kv_cache_attention: num_pages or max_pages out of range");
  TEENY_REQUIRE(num_pages * kv_heads < (int64_t{1} << 29), TEENY_ERR_SHAPE_MISMATCH,
                "kv_cache_attention: num_pages * kv_heads must be below 2^29");
  TEENY_REQUIRE(q_starts != nullptr || n_tokens == batch, TEENY_ERR_SHAPE_MISMATCH,
                "kv_cache_attention: without q_starts there is one query per sequence");
  if (n_tokens == 0 || batch == 0 || q_heads == 0) return TEENY_OK;
  TEENY_REQUIRE(q != nullptr && o != nullptr && context_lens != nullptr, TEENY_ERR_NULL_POINTER,
                "kv_cache_attention: q/o/context_lens");
  TEENY_REQUIRE((max_pages == 0 || block_table != nullptr) &&
                    (num_pages == 0 || (k_cache != nullptr && v_cache != nullptr && k_scale != nullptr && v_scale != nullptr)),
                TEENY_ERR_NULL_POINTER, "kv_cache_attention: block_table/cache/scale");
  TEENY_REQUIRE(q_stride >= q_heads * head_dim, TEENY_ERR_SHAPE_MISMATCH,
                "kv_cache_attention: token stride below q_heads * head_dim");
  TEENY_REQUIRE(aligned(q, 16) && aligned(o, 16) && aligned(k_cache, 16) && aligned(v_cache, 16) && q_stride % 8 == 0,
                TEENY_ERR_MISALIGNED, "kv_cache_attention: 16-byte aligned tensors and token stride");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const Scratch scr = stream_scratch(s);
  max_context = std::min(std::max<int64_t>(max_context, 1), std::max<int64_t>(max_pages * page_size, 1));
  const KvAttnPlan pl =
      kv_attn_plan(n_tokens, batch, q_heads, kv_heads, head_dim, max_q_len, max_context, scr.ptr ? scr.bytes : 0);
  const int64_t units = pl.blocks * kv_heads;
  TEENY_REQUIRE(units * pl.rb < (int64_t{1} << 31) / 64, TEENY_ERR_SHAPE_MISMATCH,
                "kv_cache_attention: too many rows for a launch");
  KvAttnArgs p{};
  p.q = static_cast<const bf16 *>(q);
  p.q_stride = q_stride;
  p.kc = k_cache;
  p.vc = v_cache;
  p.ks = k_scale;
  p.vs = v_scale;
  p.table = block_table;
  p.ctx = context_lens;
  p.starts = q_starts;
  p.o = static_cast<bf16 *>(o);
  p.l = l;
  p.part = pl.splits > 1 ? static_cast<float *>(scr.ptr) : nullptr;
  p.ml_off = units * pl.splits * pl.rb * head_dim;
  p.batch = static_cast<int>(batch);
  p.tokens = static_cast<int>(n_tokens);
  p.heads = static_cast<int>(q_heads);
  p.kv_heads = static_cast<int>(kv_heads);
  p.group = static_cast<int>(q_heads / kv_heads);
  p.pages = static_cast<int>(num_pages);
  p.shift = shift;
  p.width = num_pages > 0 ? static_cast<int>(max_pages) : 0;
  p.blocks = static_cast<int>(pl.blocks);
  p.walk = static_cast<int>(pl.walk);
  p.splits = pl.splits;
  p.chunk = pl.chunk;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.causal = causal != 0;
  if (head_dim == 64) launch_kv_attn<64>(pl, p, s);
  else launch_kv_attn<128>(pl, p, s);
  return after_launch(nm, s);
}

teeny_status teeny_kv_cache_attention_workspace_size(int64_t n_tokens, int64_t batch, int64_t q_heads, int64_t kv_heads,
                                                     int64_t head_dim, int64_t max_q_len, int64_t max_context,
                                                     size_t *bytes) {
  const char *nm = "kv_cache_attention_workspace_size";
  TEENY_REQUIRE(bytes != nullptr, TEENY_ERR_NULL_POINTER, "kv_cache_attention_workspace_size: bytes");
  *bytes = 0;
  teeny_status st = kv_attn_sizes(nm, n_tokens, batch, q_heads, kv_heads, head_dim, max_q_len, max_context);
  if (st != TEENY_OK) return st;
  if (n_tokens == 0 || batch == 0 || q_heads == 0) return TEENY_OK;
  *bytes = kv_attn_plan(n_tokens, batch, q_heads, kv_heads, head_dim, max_q_len, max_context, SIZE_MAX).most;
  return TEENY_OK;
}

}  // extern "C"
