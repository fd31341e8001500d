// What the attentions over the paged K/V caches (8 bits: kv_attn.hip, 4 bits: kv4_attn.hip) share: arguments, which
// rows a workgroup takes, the join of splits, and the checks of the entry points.
#pragma once

#include "mfma.hpp"

#include <algorithm>

namespace teeny {

int kv_page_shift(int64_t page_size);

struct KvAttnArgs {
  const bf16 *q;
  int64_t q_stride;
  const int8_t *kc, *vc;
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

// The same value in the four lanes l % 16, l % 16 + 16, ..: their maximum or sum.
template <typename F>
__device__ __forceinline__ float over_groups(float v, F f) {
  v = f(v, __shfl_xor(v, 16, 64));
  return f(v, __shfl_xor(v, 32, 64));
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

struct KvAttnPlan {
  bool tile = false;
  int nq = 1, rb = 16;
  int64_t blocks = 0, walk = 0;  // row blocks of a head at most; as the lengths have it
  int splits = 1, chunk = 0;
  size_t bytes = 0, most = 0;  // of workspace: used; enough for this and any smaller max_context
};

inline teeny_status kv_attn_sizes(const char *nm, int64_t n_tokens, int64_t batch, int64_t q_heads, int64_t kv_heads,
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

using KvAttnPlanFn = KvAttnPlan (*)(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t D, int64_t max_q,
                                    int64_t max_ctx, size_t scratch);

// An entry point's checks, its plan, and the arguments but for the scales.  With
// nothing to do: TEENY_OK and no blocks.
inline teeny_status kv_attn_open(const char *nm, KvAttnPlanFn plan, const void *q, const int8_t *k_cache,
                                 const int8_t *v_cache, const void *k_scale, const void *v_scale,
                                 const int32_t *block_table, const int32_t *context_lens, const int32_t *q_starts, void *o,
                                 float *l, int64_t n_tokens, int64_t batch, int64_t q_heads, int64_t kv_heads,
                                 int64_t head_dim, int64_t num_pages, int64_t page_size, int64_t max_pages,
                                 int64_t max_q_len, int64_t max_context, int64_t q_stride, float softmax_scale,
                                 int32_t causal, teeny_stream stream, KvAttnArgs &p, KvAttnPlan &pl) {
  auto at = [&](const char *msg) { return std::string(nm) + ": " + msg; };
  teeny_status st = kv_attn_sizes(nm, n_tokens, batch, q_heads, kv_heads, head_dim, max_q_len, max_context);
  if (st != TEENY_OK) return st;
  const int shift = kv_page_shift(page_size);
  TEENY_REQUIRE(shift > 0, TEENY_ERR_UNSUPPORTED, at("page_size must be 16, 32, 64 or 128"));
  TEENY_REQUIRE(num_pages >= 0 && max_pages >= 0 && num_pages <= 0x7fffffff / page_size &&
                    max_pages <= (0x7fffffff - 4096) / page_size,
                TEENY_ERR_SHAPE_MISMATCH, at("num_pages or max_pages out of range"));
  TEENY_REQUIRE(num_pages * kv_heads < (int64_t{1} << 29), TEENY_ERR_SHAPE_MISMATCH,
                at("num_pages * kv_heads must be below 2^29"));
  TEENY_REQUIRE(q_starts != nullptr || n_tokens == batch, TEENY_ERR_SHAPE_MISMATCH,
                at("without q_starts there is one query per sequence"));
  pl.blocks = 0;
  if (n_tokens == 0 || batch == 0 || q_heads == 0) return TEENY_OK;
  TEENY_REQUIRE(q != nullptr && o != nullptr && context_lens != nullptr, TEENY_ERR_NULL_POINTER, at("q/o/context_lens"));
  TEENY_REQUIRE((max_pages == 0 || block_table != nullptr) &&
                    (num_pages == 0 || (k_cache != nullptr && v_cache != nullptr && k_scale != nullptr && v_scale != nullptr)),
                TEENY_ERR_NULL_POINTER, at("block_table/cache/scale"));
  TEENY_REQUIRE(q_stride >= q_heads * head_dim, TEENY_ERR_SHAPE_MISMATCH, at("token stride below q_heads * head_dim"));
  TEENY_REQUIRE(aligned(q, 16) && aligned(o, 16) && aligned(k_cache, 16) && aligned(v_cache, 16) && q_stride % 8 == 0,
                TEENY_ERR_MISALIGNED, at("16-byte aligned tensors and token stride"));
  const Scratch scr = stream_scratch(static_cast<hipStream_t>(stream));
  max_context = std::min(std::max<int64_t>(max_context, 1), std::max<int64_t>(max_pages * page_size, 1));
  pl = plan(n_tokens, batch, q_heads, kv_heads, head_dim, max_q_len, max_context, scr.ptr ? scr.bytes : 0);
  const int64_t units = pl.blocks * kv_heads;
  // a join has 64 threads for each row; 256 threads to a row block, 512 to one of 256 rows, leave room for four splits
  TEENY_REQUIRE(units * std::min(pl.rb, 128) < (int64_t{1} << 31) / 64 && n_tokens * q_heads < (int64_t{1} << 31) / 64,
                TEENY_ERR_SHAPE_MISMATCH, at("too many rows for a launch"));
  p.q = static_cast<const bf16 *>(q);
  p.q_stride = q_stride;
  p.kc = k_cache;
  p.vc = v_cache;
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
  return TEENY_OK;
}

inline teeny_status kv_attn_workspace(const char *nm, KvAttnPlanFn plan, int64_t n_tokens, int64_t batch, int64_t q_heads,
                                      int64_t kv_heads, int64_t head_dim, int64_t max_q_len, int64_t max_context,
                                      size_t *bytes) {
  TEENY_REQUIRE(bytes != nullptr, TEENY_ERR_NULL_POINTER, std::string(nm) + ": bytes");
  *bytes = 0;
  teeny_status st = kv_attn_sizes(nm, n_tokens, batch, q_heads, kv_heads, head_dim, max_q_len, max_context);
  if (st != TEENY_OK) return st;
  if (n_tokens == 0 || batch == 0 || q_heads == 0) return TEENY_OK;
  *bytes = plan(n_tokens, batch, q_heads, kv_heads, head_dim, max_q_len, max_context, SIZE_MAX).most;
  return TEENY_OK;
}

}  // namespace teeny
